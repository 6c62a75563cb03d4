"""The evaluator behind the reference's ``Network`` trait (src/net/mod.rs:264-296), in Python.

``B200Network`` is the drop-in for ``CudaNetwork`` (src/net/cuda/mod.rs:225-1012): it
owns one library context (``mrn_ctx``) on one GPU, packs leaves the way the reference's CUDA
backend does (src/net/cuda/mod.rs:946-967) and slices each position's priors out of the
224-slot output (:994-999). ``GroupNetwork`` implements the same trait over several GPUs
through the library's own multi-device evaluator (``mrn_group_*``: contiguous shards, one
per GPU, evaluated at the same time by native per-device threads and written back in
order); ``ShardedNetwork`` does the same from Python threads over any replicas. No
collective is involved: the positions are independent. Errors surface as ``NetworkError``; nothing is ever substituted for a
network's answer (src/net/mod.rs:284-288).
"""

from __future__ import annotations

import ctypes
import threading
from abc import ABC, abstractmethod
from concurrent.futures import ThreadPoolExecutor
from ctypes import POINTER, c_double, c_float, c_int, c_int32, c_uint8, c_void_p
from dataclasses import dataclass
from typing import Sequence

import numpy as np

from . import _lib
from .model import Architecture
from .weights import Weights

MAX_LEGAL = _lib.MAX_LEGAL
BOARD_BYTES = _lib.BOARD_BYTES


class NetworkError(RuntimeError):
    """A backend that can no longer evaluate (`NetworkError`, src/net/mod.rs:284-288)."""

    def __init__(self, message: str, code: int = 0):
        super().__init__(message)
        self.code = code


@dataclass
class Evaluation:
    """What the network says about one position, from the side to move
    (src/net/mod.rs:264-279)."""

    priors: np.ndarray  # one prior per legal move, in the leaf's move order, summing to 1
    wdl: tuple[float, float, float]

    def value(self) -> float:
        return self.wdl[0] - self.wdl[2]


# A leaf: (66-byte encoded board, legal action indices in move order), the packed form of
# the reference's `Leaf = (&EncodedBoard, &LegalActions)` (src/net/mod.rs:281-282).
Leaf = tuple


class Network(ABC):
    @abstractmethod
    def evaluate(self, batch: Sequence[Leaf]) -> list[Evaluation]:
        """One `Evaluation` per input, in order; priors cover exactly the legal moves."""

    @abstractmethod
    def describe(self) -> str:
        """Human-readable description for `info string` at load time."""


def pack(batch: Sequence[Leaf]) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
    """Boards [n, 66] uint8, legal [n, 224] int32 (-1 padded) and move counts, as
    `CudaNetwork::forward` packs its pinned buffers (src/net/cuda/mod.rs:946-967)."""
    n = len(batch)
    boards = np.zeros((n, BOARD_BYTES), dtype=np.uint8)
    legal = np.full((n, MAX_LEGAL), -1, dtype=np.int32)
    counts = np.zeros(n, dtype=np.int32)
    for p, (board, actions) in enumerate(batch):
        boards[p] = np.frombuffer(bytes(board), dtype=np.uint8) if not isinstance(board, np.ndarray) else board
        acts = np.asarray(actions, dtype=np.int64)
        if len(acts) > MAX_LEGAL:
            raise NetworkError(f"position with {len(acts)} legal moves exceeds MAX_LEGAL {MAX_LEGAL}",
                               code=4)
        legal[p, :len(acts)] = acts
        counts[p] = len(acts)
    return boards, legal, counts


def unpack(priors: np.ndarray, wdl: np.ndarray, counts: np.ndarray) -> list[Evaluation]:
    return [Evaluation(priors[p, :counts[p]].copy(), (float(wdl[p, 0]), float(wdl[p, 1]), float(wdl[p, 2])))
            for p in range(len(counts))]


def _f32p(a: np.ndarray):
    return a.ctypes.data_as(POINTER(c_float))


def c_weights(w: Weights):
    """(mrn_weights, mrn_layer array) pointing into `w`'s arrays (keep `w` alive)."""
    L = _lib.MrnLinear
    N = _lib.MrnNorm
    lin = lambda wn, bn: L(w.ptr(wn), w.ptr(bn))  # noqa: E731
    nrm = lambda p: N(w.ptr(p + ".weight"), w.ptr(p + ".bias"))  # noqa: E731
    layers = (_lib.MrnLayer * w.arch.n_layers)()
    for i in range(w.arch.n_layers):
        p = f"encoder.layers.{i}."
        layers[i] = _lib.MrnLayer(
            nrm(p + "norm1"), lin(p + "self_attn.in_proj_weight", p + "self_attn.in_proj_bias"),
            lin(p + "self_attn.out_proj.weight", p + "self_attn.out_proj.bias"), nrm(p + "norm2"),
            lin(p + "linear1.weight", p + "linear1.bias"), lin(p + "linear2.weight", p + "linear2.bias"))
    cw = _lib.MrnWeights(
        w.ptr("piece_embed.weight"), w.ptr("square_embed.weight"), w.ptr("state_embed"),
        lin("castling_proj.weight", "castling_proj.bias"), w.ptr("en_passant_embed.weight"),
        ctypes.cast(layers, POINTER(_lib.MrnLayer)), nrm("final_norm"), nrm("policy_head.norm"),
        lin("policy_head.proj.weight", "policy_head.proj.bias"), nrm("value_head.norm"),
        lin("value_head.ff.0.weight", "value_head.ff.0.bias"), lin("value_head.ff.2.weight", "value_head.ff.2.bias"))
    return cw, layers


def c_arch(arch: Architecture):
    amax = None
    if arch.fp8_amax is not None:
        amax = np.ascontiguousarray(np.asarray(arch.fp8_amax, dtype=np.float32).reshape(-1))
    ca = _lib.MrnArch(arch.d_model, arch.n_layers, arch.n_heads, arch.d_ff, arch.layer_norm_eps, arch.gelu,
                      arch.tokens, arch.square_token_start, _f32p(amax) if amax is not None else None)
    return ca, amax


class LogitRules(_lib.MrnRules):
    """What changes the logits of a batch of rows (`mrn_rules`): device pointers as integers, 0 or
    None where a part is not used, with the lengths and strides that go with them. It holds no
    reference to the memory; keep that alive while calls with the rules are in flight."""

    def __init__(self, actions: int, **parts):
        super().__init__(actions=actions)
        for name, value in parts.items():
            if name not in _RULE_PARTS:
                raise TypeError(f"LogitRules has no part {name!r}: one of {sorted(_RULE_PARTS)}")
            setattr(self, name, value)


_RULE_PARTS = {name for name, _ in _lib.MrnRules._fields_} - {"actions"}


class MoveRules:
    """`LogitRules` in host memory, for a batch of positions' move lists (`evaluate_moves`,
    `choose_moves`); every part is optional and an array with one row is shared by the batch:

    * ``mask`` [n or 1, 4672] bool: the actions that may be played;
    * ``bias`` (actions [n or 1, k], values [n or 1, k]): added to the logits of those actions, -1
      where a list is shorter;
    * ``history`` [n or 1, h]: actions played before, -1 where a list is shorter, which ``repetition``,
      ``presence`` and ``frequency`` (a number, or one per position) make less likely. Without a history
      there is nothing that they change.
    """

    def __init__(self, mask=None, bias=None, history=None, repetition=None, presence=None, frequency=None):
        self.mask, self.bias, self.history = mask, bias, history
        self.penalties = {"repetition": repetition, "presence": presence, "frequency": frequency}

    def packed(self, n: int) -> LogitRules:
        parts, keep = {}, []

        def rows(name, value, dtype, width=None):
            a = np.ascontiguousarray(value, dtype=dtype)
            if a.ndim != 2 or a.shape[0] not in (1, n) or (width is not None and a.shape[1] != width):
                raise ValueError(f"{name} has shape {list(a.shape)}: expected [{n} or 1, {width or 'entries'}]")
            return a

        def put(name, a, stride=None):
            keep.append(a)
            parts[name] = a.ctypes.data
            if stride is not None:
                parts[stride] = 0 if a.shape[0] == 1 else a.shape[1]

        if self.mask is not None:
            allowed = rows("mask", self.mask, np.bool_, _lib.ACTIONS)
            put("mask", np.packbits(allowed, axis=1, bitorder="little").view(np.uint32), "mask_stride")
        if self.bias is not None:
            ids, values = rows("bias actions", self.bias[0], np.int32), rows("bias values", self.bias[1], np.float32)
            if ids.shape != values.shape:
                raise ValueError(f"bias actions {list(ids.shape)} and values {list(values.shape)} differ in shape")
            if ids.shape[1]:
                put("bias_actions", ids, "bias_stride")
                put("bias_values", values)
                parts["bias_len"] = ids.shape[1]
        penalties = {name: _per_row(name, value, np.float32, n) for name, value in self.penalties.items()
                     if value is not None}
        if self.history is not None:
            played = rows("history", self.history, np.int32)
            if played.shape[1]:
                put("history", played, "history_stride")
                parts["history_len"] = played.shape[1]
            for name, value in penalties.items():
                put(name, value)
        rules = LogitRules(_lib.ACTIONS, **parts)
        rules.arrays = keep
        return rules


def _per_row(name, value, dtype, n: int):
    """A number, or one per position, as a C array of n; None stays None."""
    if value is None:
        return None
    a = np.asarray(value, dtype=dtype)
    if a.shape not in ((), (n,)):
        raise ValueError(f"{name} has shape {list(a.shape)}: expected a number or [{n}]")
    return np.ascontiguousarray(np.broadcast_to(a, (n,)))


def _data(a):
    return None if a is None else a.ctypes.data


def _move_lists(boards, lengths, actions):
    boards = np.ascontiguousarray(boards, dtype=np.uint8)
    lengths = np.ascontiguousarray(lengths, dtype=np.int32)
    actions = np.ascontiguousarray(actions, dtype=np.int32)
    n = boards.shape[0]
    if boards.shape != (n, BOARD_BYTES) or lengths.shape != (n,) or actions.ndim != 1:
        raise ValueError("boards must be [n, 66], lengths [n] and actions one list")
    if (lengths < 0).any() or int(lengths.sum(dtype=np.int64)) != len(actions):
        raise ValueError(f"lengths add up to {int(lengths.sum(dtype=np.int64))}, actions hold {len(actions)}")
    return n, boards, lengths, actions


class B200Network(Network):
    """One GPU's evaluator: `CudaNetwork::new(arch, &weights, ordinal, max_batch, fp8)`
    (src/net/cuda/mod.rs:276-493) with `precision` one of "bf16", "fp8w" (e4m3 weights,
    bf16 activations), "fp8" (e4m3 weights and activations) or "fp8x2" (e4m3 weights,
    activations as two e4m3 terms each)."""

    def __init__(self, arch: Architecture, weights: Weights, device: int = 0, max_batch: int = 1024,
                 precision: str = "fp8w"):
        self._lib = _lib.load()
        if precision not in _lib.PRECISIONS:
            raise ValueError(f"precision {precision!r}: one of {sorted(_lib.PRECISIONS)}")
        self.arch, self.device, self.max_batch, self.precision = arch, device, max_batch, precision
        ca, amax = c_arch(arch)
        cw, layers = c_weights(weights)
        ctx = c_void_p()
        rc = self._lib.mrn_create(ctypes.byref(ca), ctypes.byref(cw), device, max_batch,
                                  _lib.PRECISIONS[precision], ctypes.byref(ctx))
        del amax, layers
        if rc != 0:
            raise NetworkError(f"b200 backend failed to load: {self._lib.mrn_last_error(None).decode()}", rc)
        self._ctx = ctx
        self._lock = threading.Lock()

    # -- the trait --------------------------------------------------------------------------
    def evaluate(self, batch: Sequence[Leaf]) -> list[Evaluation]:
        boards, legal, counts = pack(batch)
        priors, wdl = self.evaluate_packed(boards, legal)
        return unpack(priors, wdl, counts)

    def describe(self) -> str:
        return self._lib.mrn_describe(self._ctx).decode()

    # -- packed / raw entry points ---------------------------------------------------------
    def _check(self, rc: int, what: str):
        if rc != 0:
            raise NetworkError(f"b200 {what} failed: {self._lib.mrn_last_error(self._ctx).decode()}", rc)

    def evaluate_packed(self, boards: np.ndarray, legal: np.ndarray, priors: np.ndarray | None = None,
                        wdl: np.ndarray | None = None) -> tuple[np.ndarray, np.ndarray]:
        """`mrn_evaluate` on packed host arrays: boards [n, 66] uint8, legal [n, 224] int32.
        Returns priors [n, 224] and wdl [n, 3] (written into `priors` / `wdl` when given)."""
        boards = np.ascontiguousarray(boards, dtype=np.uint8)
        legal = np.ascontiguousarray(legal, dtype=np.int32)
        n = boards.shape[0]
        if boards.shape != (n, BOARD_BYTES) or legal.shape != (n, MAX_LEGAL):
            raise ValueError("boards must be [n, 66] and legal [n, 224]")
        if priors is None:
            priors = np.empty((n, MAX_LEGAL), dtype=np.float32)
        if wdl is None:
            wdl = np.empty((n, 3), dtype=np.float32)
        rc = self._lib.mrn_evaluate(self._ctx, n, boards.ctypes.data_as(POINTER(c_uint8)),
                                    legal.ctypes.data_as(POINTER(c_int32)), _f32p(priors), _f32p(wdl))
        self._check(rc, "forward")
        return priors, wdl

    def evaluate_packed_f16(self, boards: np.ndarray, legal: np.ndarray, priors: np.ndarray | None = None,
                            wdl: np.ndarray | None = None) -> tuple[np.ndarray, np.ndarray]:
        """`mrn_evaluate_f16`: as `evaluate_packed`, with the priors returned as float16 [n, 224]
        (half the bytes copied back from the GPU; written into `priors` / `wdl` when given)."""
        boards = np.ascontiguousarray(boards, dtype=np.uint8)
        legal = np.ascontiguousarray(legal, dtype=np.int32)
        n = boards.shape[0]
        if boards.shape != (n, BOARD_BYTES) or legal.shape != (n, MAX_LEGAL):
            raise ValueError("boards must be [n, 66] and legal [n, 224]")
        if priors is None:
            priors = np.empty((n, MAX_LEGAL), dtype=np.float16)
        if wdl is None:
            wdl = np.empty((n, 3), dtype=np.float32)
        if priors.dtype != np.float16 or priors.shape != (n, MAX_LEGAL) or not priors.flags.c_contiguous:
            raise ValueError("priors must be a C-contiguous float16 [n, 224] array")
        rc = self._lib.mrn_evaluate_f16(self._ctx, n, boards.ctypes.data_as(POINTER(c_uint8)),
                                        legal.ctypes.data_as(POINTER(c_int32)), priors.ctypes.data, _f32p(wdl))
        self._check(rc, "forward")
        return priors, wdl

    def logits(self, boards: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
        """Raw policy logits [n, 4672] and WDL logits [n, 3] (`CpuNetwork::logits`)."""
        boards = np.ascontiguousarray(boards, dtype=np.uint8)
        n = boards.shape[0]
        policy = np.empty((n, _lib.ACTIONS), dtype=np.float32)
        value = np.empty((n, 3), dtype=np.float32)
        rc = self._lib.mrn_logits(self._ctx, n, boards.ctypes.data_as(POINTER(c_uint8)), _f32p(policy), _f32p(value))
        self._check(rc, "logits")
        return policy, value

    def evaluate_device(self, n: int, boards_ptr: int, legal_ptr: int, priors_ptr: int, wdl_ptr: int,
                        stream: int | None = None) -> None:
        """Enqueue a forward pass on device-resident buffers (device pointers) on `stream`."""
        rc = self._lib.mrn_evaluate_device(self._ctx, n, c_void_p(boards_ptr), c_void_p(legal_ptr),
                                           c_void_p(priors_ptr), c_void_p(wdl_ptr), c_void_p(stream or 0))
        self._check(rc, "device forward")

    def evaluate_device_static(self, n: int, boards_ptr: int, legal_ptr: int, priors_ptr: int, wdl_ptr: int,
                               stream: int | None = None) -> None:
        """`evaluate_device` without any device allocation: the pass's intermediates live in the
        library's static 8 MiB device array, so it serves callers that must not allocate once
        running, for small batches (see `mrn_evaluate_device_static`). Calls whose GPU work
        overlaps share that array and race; serialise them."""
        rc = self._lib.mrn_evaluate_device_static(self._ctx, n, c_void_p(boards_ptr), c_void_p(legal_ptr),
                                                  c_void_p(priors_ptr), c_void_p(wdl_ptr), c_void_p(stream or 0))
        self._check(rc, "static-scratch forward")

    # -- move lists ---------------------------------------------------------------------------
    def evaluate_moves(self, boards: np.ndarray, lengths: np.ndarray, actions: np.ndarray,
                       rules: MoveRules | None = None, temperature=None) -> tuple[np.ndarray, np.ndarray]:
        """`mrn_evaluate_moves`: boards [n, 66], lengths [n] and the positions' legal actions one list
        behind the other. Returns a prior for each listed action, in the same order, under `rules` and
        at `temperature` (a number or one per position), and wdl [n, 3]."""
        n, boards, lengths, actions = _move_lists(boards, lengths, actions)
        packed = None if rules is None else rules.packed(n)
        t = _per_row("temperature", temperature, np.float32, n)
        priors = np.empty(len(actions), dtype=np.float32)
        wdl = np.empty((n, 3), dtype=np.float32)
        rc = self._lib.mrn_evaluate_moves(self._ctx, n, _data(boards), _data(lengths), _data(actions), packed, _data(t),
                                          _data(priors), _data(wdl))
        self._check(rc, "forward on move lists")
        return priors, wdl

    def choose_moves(self, boards: np.ndarray, lengths: np.ndarray, actions: np.ndarray, uniform=None,
                     rules: MoveRules | None = None, temperature=None, top_k=None,
                     top_p=None) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
        """`mrn_choose_moves`: one move per position, drawn with `uniform` (numbers in [0, 1), one per
        position; None: the likeliest move). Returns the move's place in its position's list (-1: none
        is left), its probability and wdl [n, 3]."""
        n, boards, lengths, actions = _move_lists(boards, lengths, actions)
        packed = None if rules is None else rules.packed(n)
        t, u = _per_row("temperature", temperature, np.float32, n), _per_row("uniform", uniform, np.float32, n)
        k, p = _per_row("top_k", top_k, np.int32, n), _per_row("top_p", top_p, np.float32, n)
        move, prob = np.empty(n, dtype=np.int32), np.empty(n, dtype=np.float32)
        wdl = np.empty((n, 3), dtype=np.float32)
        rc = self._lib.mrn_choose_moves(self._ctx, n, _data(boards), _data(lengths), _data(actions), packed, _data(t),
                                        _data(k), _data(p), _data(u), _data(move), _data(prob), _data(wdl))
        self._check(rc, "choice of moves")
        return move, prob, wdl

    # -- policy operators (device pointers; enqueued on `stream`, the context's own if None) -----
    def slot_table(self, rows: int, width: int, lengths_ptr: int, count: int, entries_ptr: int, starts_ptr: int,
                   table_ptr: int, map_ptr: int | None = None, stream: int | None = None) -> None:
        """`mrn_slot_table`: `rows` lists laid one behind the other in `entries` (int32, `count` in all)
        into slot rows of `width`, -1 behind each list; `starts` [rows + 1] and the slot of each entry
        in `map` [count], all int32."""
        rc = self._lib.mrn_slot_table(self._ctx, rows, width, lengths_ptr, count, entries_ptr, starts_ptr, table_ptr,
                                      map_ptr, stream)
        self._check(rc, "slot table")

    def adjust_logits(self, rows: int, width: int, logits_ptr: int, rules: LogitRules | None = None,
                      out_ptr: int | None = None, priors_ptr: int | None = None, dtype: str = "f32",
                      stride: int | None = None, out_stride: int | None = None, priors_stride: int | None = None,
                      temperature_ptr: int | None = None, stream: int | None = None) -> None:
        """`mrn_adjust_logits`: the logits (`dtype` "f32", "f16" or "bf16") under `rules` into `out` (the
        same type; may be the logits themselves) and their softmax at each row's temperature into
        `priors` (f32). Strides are in elements, `width` where not given."""
        if dtype not in _lib.TYPES:
            raise ValueError(f"dtype {dtype!r}: one of {sorted(_lib.TYPES)}")
        rc = self._lib.mrn_adjust_logits(self._ctx, rows, width, logits_ptr, _lib.TYPES[dtype],
                                         width if stride is None else stride, rules, temperature_ptr, out_ptr,
                                         width if out_stride is None else out_stride, priors_ptr,
                                         width if priors_stride is None else priors_stride, stream)
        self._check(rc, "adjust logits")

    def choose_actions(self, rows: int, width: int, logits_ptr: int, rules: LogitRules | None, column_ptr: int,
                       action_ptr: int | None = None, prob_ptr: int | None = None, dtype: str = "f32",
                       stride: int | None = None, temperature_ptr: int | None = None, top_k_ptr: int | None = None,
                       top_p_ptr: int | None = None, uniform_ptr: int | None = None, stream: int | None = None) -> None:
        """`mrn_choose_actions`: one column per row (int32, -1 where nothing is left), its action (int32)
        and its share of the kept mass (f32), drawn with `uniform` [rows] from the logits under `rules`
        at each row's temperature, within `top_k` (int32) and `top_p` (f32)."""
        if dtype not in _lib.TYPES:
            raise ValueError(f"dtype {dtype!r}: one of {sorted(_lib.TYPES)}")
        rc = self._lib.mrn_choose_actions(self._ctx, rows, width, logits_ptr, _lib.TYPES[dtype],
                                          width if stride is None else stride, rules, temperature_ptr, top_k_ptr,
                                          top_p_ptr, uniform_ptr, column_ptr, action_ptr, prob_ptr, stream)
        self._check(rc, "choose actions")

    def status_word(self) -> int:
        word = c_int()
        self._check(self._lib.mrn_status_word(self._ctx, ctypes.byref(word)), "status")
        return word.value

    def profile(self, n: int, boards_ptr: int, legal_ptr: int, priors_ptr: int, wdl_ptr: int,
                stream: int | None = None) -> dict:
        """Per kernel class: device ms, algorithmic FLOPs and launches of one eager pass."""
        k = len(_lib.PROFILE_SLOTS)
        times = (c_float * k)()
        flops = (c_double * k)()
        launches = (c_int * k)()
        rc = self._lib.mrn_profile(self._ctx, n, c_void_p(boards_ptr), c_void_p(legal_ptr), c_void_p(priors_ptr),
                                   c_void_p(wdl_ptr), c_void_p(stream or 0), times, flops, launches)
        self._check(rc, "profile")
        return {name: {"ms": times[i], "flops": flops[i], "launches": launches[i]}
                for i, name in enumerate(_lib.PROFILE_SLOTS)}

    def launches_per_forward(self, n: int) -> int:
        return int(self._lib.mrn_launches_per_forward(self._ctx, n))

    def close(self) -> None:
        if getattr(self, "_ctx", None):
            self._lib.mrn_destroy(self._ctx)
            self._ctx = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class GroupNetwork(Network):
    """`Network` over one weight replica per listed device through `mrn_group_create` /
    `mrn_group_evaluate`: every batch is cut into contiguous shards (sizes differing by at most
    one position), evaluated at the same time by the library's per-device threads and written
    into the outputs in input order. A batch larger than `max_batch` runs as consecutive
    `max_batch` chunks whose shards the threads take as they become free. A failing shard raises
    `NetworkError` naming its device and positions."""

    def __init__(self, arch: Architecture, weights: Weights, devices: Sequence[int], max_batch: int = 1024,
                 precision: str = "fp8w"):
        self._lib = _lib.load()
        if precision not in _lib.PRECISIONS:
            raise ValueError(f"precision {precision!r}: one of {sorted(_lib.PRECISIONS)}")
        self.arch, self.devices, self.max_batch, self.precision = arch, list(devices), max_batch, precision
        ca, amax = c_arch(arch)
        cw, layers = c_weights(weights)
        devs = (c_int * len(self.devices))(*self.devices)
        group = c_void_p()
        rc = self._lib.mrn_group_create(ctypes.byref(ca), ctypes.byref(cw), devs, len(self.devices), max_batch,
                                        _lib.PRECISIONS[precision], ctypes.byref(group))
        del amax, layers
        if rc != 0:
            raise NetworkError(f"b200 group failed to load: {self._lib.mrn_group_last_error(None).decode()}", rc)
        self._group = group

    def evaluate(self, batch: Sequence[Leaf]) -> list[Evaluation]:
        boards, legal, counts = pack(batch)
        priors, wdl = self.evaluate_packed(boards, legal)
        return unpack(priors, wdl, counts)

    def evaluate_packed(self, boards: np.ndarray, legal: np.ndarray, priors: np.ndarray | None = None,
                        wdl: np.ndarray | None = None) -> tuple[np.ndarray, np.ndarray]:
        """`mrn_group_evaluate` on packed host arrays (see `B200Network.evaluate_packed`)."""
        boards = np.ascontiguousarray(boards, dtype=np.uint8)
        legal = np.ascontiguousarray(legal, dtype=np.int32)
        n = boards.shape[0]
        if boards.shape != (n, BOARD_BYTES) or legal.shape != (n, MAX_LEGAL):
            raise ValueError("boards must be [n, 66] and legal [n, 224]")
        if priors is None:
            priors = np.empty((n, MAX_LEGAL), dtype=np.float32)
        if wdl is None:
            wdl = np.empty((n, 3), dtype=np.float32)
        rc = self._lib.mrn_group_evaluate(self._group, n, boards.ctypes.data_as(POINTER(c_uint8)),
                                          legal.ctypes.data_as(POINTER(c_int32)), _f32p(priors), _f32p(wdl))
        if rc != 0:
            raise NetworkError(f"b200 group forward failed: {self._lib.mrn_group_last_error(self._group).decode()}",
                               rc)
        return priors, wdl

    def describe(self) -> str:
        return self._lib.mrn_group_describe(self._group).decode()

    def close(self) -> None:
        if getattr(self, "_group", None):
            self._lib.mrn_group_destroy(self._group)
            self._group = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class ShardedNetwork(Network):
    """`Network` over one replica per GPU: each batch is cut into contiguous shards (one per
    replica, sizes differing by at most one), evaluated concurrently by per-GPU evaluator
    threads, and concatenated in order. The first shard error is raised as `NetworkError`."""

    def __init__(self, replicas: Sequence[Network]):
        if not replicas:
            raise ValueError("no replicas")
        self.replicas = list(replicas)
        self._pool = ThreadPoolExecutor(max_workers=len(self.replicas), thread_name_prefix="marina-b200-gpu")

    @staticmethod
    def shards(n: int, k: int) -> list[tuple[int, int]]:
        base, extra = divmod(n, k)
        out, start = [], 0
        for i in range(k):
            size = base + (1 if i < extra else 0)
            out.append((start, start + size))
            start += size
        return out

    def evaluate(self, batch: Sequence[Leaf]) -> list[Evaluation]:
        spans = [s for s in self.shards(len(batch), len(self.replicas))]
        futures = [self._pool.submit(r.evaluate, batch[a:b]) for r, (a, b) in zip(self.replicas, spans) if b > a]
        out: list[Evaluation] = []
        error = None
        for f in futures:
            try:
                out.extend(f.result())
            except Exception as e:  # noqa: BLE001 - re-raised below as the trait's error type
                error = error or e
        if error is not None:
            raise error if isinstance(error, NetworkError) else NetworkError(str(error))
        return out

    def _packed(self, method: str, prior_dtype, boards: np.ndarray, legal: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
        """Packed batches: each replica writes its shard straight into its rows of the outputs."""
        n = boards.shape[0]
        priors = np.empty((n, MAX_LEGAL), dtype=prior_dtype)
        wdl = np.empty((n, 3), dtype=np.float32)
        spans = self.shards(n, len(self.replicas))
        futures = [self._pool.submit(getattr(r, method), boards[a:b], legal[a:b], priors[a:b], wdl[a:b])
                   for r, (a, b) in zip(self.replicas, spans) if b > a]
        error = None
        for f in futures:
            try:
                f.result()
            except Exception as e:  # noqa: BLE001 - re-raised below as the trait's error type
                error = error or e
        if error is not None:
            raise error if isinstance(error, NetworkError) else NetworkError(str(error))
        return priors, wdl

    def evaluate_packed(self, boards: np.ndarray, legal: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
        return self._packed("evaluate_packed", np.float32, boards, legal)

    def evaluate_packed_f16(self, boards: np.ndarray, legal: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
        return self._packed("evaluate_packed_f16", np.float16, boards, legal)

    def describe(self) -> str:
        return f"{len(self.replicas)} replicas: " + "; ".join(r.describe() for r in self.replicas)
