"""Mixture-of-experts operators: routing, slot map, grouped products, combine, and their
backward passes (``csrc/kernels/expert_*.cu``).

A layer runs them in this order::

    weights, ids = route_experts(logits, top_k)            # [tokens, top_k]
    slots = expert_slots(ids, num_experts)                 # (token, choice) pairs by expert
    h = expert_gemm(x, w_gate_up, slots, epilogue="silu_gate")
    y = expert_gemm(h, w_down, slots, rows="slots")
    out = expert_combine(y, slots, weights)                # [tokens, hidden]

Nothing here synchronises with the host: how many rows an expert has stays on the GPU, and
every shape depends on ``tokens * top_k`` alone, so a layer can be captured into a CUDA graph.
All results repeat bit for bit from call to call.  The functions record no autograd graph; each
``*_backward`` takes what its forward function took.

``stream``: the stream to run on (default: the current stream of the tensors' device).  Results
are allocated on that stream; the caller orders it behind the work that produced the inputs.
"""

from __future__ import annotations

import ctypes as C
import threading
from dataclasses import dataclass
from functools import lru_cache
from typing import Optional

import torch

from .. import _native
from . import fused_gemm as _fg

MAX_ROUTED_EXPERTS = 512
MAX_EXPERTS = 1024
MAX_TOP_K = 32

_LOGIT_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_EPILOGUES = {"none": 0, "silu_gate": 1}
_EPI_SILU_GATE_GRAD, _EPI_FLOAT = 2, 3
_SCORES = {"softmax": 0, "sigmoid": 1}
_GROUP_SCORES = {"top2": 0, "max": 1}
_ROWS = ("tokens", "slots")


# --------------------------------------------------------------------------- checks
def _choice(name: str, value, table):
    if value not in table:
        raise ValueError(f"{name} must be one of {tuple(table)}, got {value!r}")
    return table[value] if isinstance(table, dict) else value


def _check_tensor(name: str, t, dim: int, dtypes, device=None, *, contiguous: bool = False):
    if not isinstance(t, torch.Tensor) or t.dim() != dim:
        raise ValueError(f"{name} must be a {dim}-D tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must have dtype {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if contiguous and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t


def _pitch(name: str, t) -> int:
    """Elements between rows of a row-major matrix (the last two dimensions of ``t``)."""
    if t.stride(-1) != 1 and t.shape[-1] != 1:
        raise ValueError(f"{name} must be row-major with unit column stride")
    if t.shape[-2] <= 1:
        return t.shape[-1]
    if t.stride(-2) < t.shape[-1]:
        raise ValueError(f"{name} has rows that overlap (row stride {t.stride(-2)}, "
                         f"{t.shape[-1]} columns)")
    return t.stride(-2)


_HALF = (torch.float16, torch.bfloat16)


# The raw handle of a device's current stream and the current device, without the Python objects
# around them (a microsecond of a call's fourteen).
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") \
    else lambda index: torch.cuda.current_stream(index).cuda_stream
_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") \
    else torch.cuda.current_device


class _Elsewhere:
    """Makes another device or stream than the current one current; inputs used on ``stream``
    are reported to the caching allocator."""

    def __init__(self, dev, stream, inputs):
        self.guards = [torch.cuda.device(dev)]
        if stream is not None:
            if stream.device != dev:
                raise ValueError(f"stream is on {stream.device}, the tensors are on {dev}")
            for t in inputs:
                if t is not None:
                    t.record_stream(stream)
            self.guards.append(torch.cuda.stream(stream))
        for g in self.guards:
            g.__enter__()

    def leave(self) -> None:
        for g in reversed(self.guards):
            g.__exit__(None, None, None)


def _enter(stream, *inputs):
    """``(raw stream, guard)`` of a call on ``inputs``' device; the guard is None in the common
    case that device and stream are current, and otherwise left when the call is done."""
    index = inputs[0].get_device()
    if index < 0:
        raise ValueError(f"the expert operators take CUDA tensors, got tensors on {inputs[0].device}")
    guard = None
    if stream is not None or _current_device() != index:
        guard = _Elsewhere(inputs[0].device, stream, inputs)
    return _raw_stream(index), guard


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


_ENTRIES: dict = {}


def _launch(fn: str, *args) -> None:
    entry = _ENTRIES.get(fn)
    if entry is None:
        entry = getattr(_native.load(), fn, None)
        if entry is None:
            raise _native.NativeError(fn, -1, "symbol not present in this build of libtileccl_b200")
        _ENTRIES[fn] = entry
    rc = entry(*args)
    if rc != 0:
        _native.check(fn, rc)
    _fg.count_launches(1)


# Held while per-device state is made or handed out: host threads may make their first calls together.
_STATE_LOCK = threading.Lock()

_STATUS: dict = {}                        # device index -> address of its status words
_ARENAS: dict = {}                        # device index -> its _CounterArena


class _CounterArena:
    """Zeroed arrival counters of one device's products.  Every call leaves its counters at zero.
    Calls on one stream follow one another and share a piece; a captured call gets a piece of its
    own for good, because its graph may be replayed beside anything else."""

    def __init__(self, address: int, nbytes: int):
        self.address, self.BYTES = address, nbytes        # (some 800 pieces)
        self.used, self.by_stream = 0, {}

    def take(self, nbytes: int) -> int:
        """Address of a new piece, 0 when none is left (under the lock: no piece is given twice)."""
        at = self.used
        if at + nbytes > self.BYTES:
            return 0
        self.used = at + -(-nbytes // 128) * 128
        return self.address + at


def _device_state(index: int) -> None:
    """Looks up the status words and counters of the current device, ``index`` (under the lock)."""
    status, counters, nbytes = C.c_uint64(), C.c_uint64(), C.c_int64()
    _native.call("tccl_expert_state", C.byref(status), C.byref(counters), C.byref(nbytes))
    _ARENAS[index] = _CounterArena(counters.value, nbytes.value)
    _STATUS[index] = status.value


def _status_ptr(dev: torch.device) -> int:
    """Status words of a device's products (see :func:`check_expert_status`)."""
    address = _STATUS.get(dev.index)
    if address is None:
        with _STATE_LOCK:
            if dev.index not in _STATUS:
                _device_state(dev.index)
            address = _STATUS[dev.index]
    return address


_MIN_BUDGET_NS = 2_000_000_000


def _wait_budget_ns() -> int:
    """Budget of a product's waits.  They wait for the kernel's own copies and products, never for
    a peer, so ``TILECCL_WAIT_BUDGET_US`` can only lengthen them: a budget that suits peers would
    end long products that nothing is wrong with."""
    return max(_fg._config().wait_budget_ns, _MIN_BUDGET_NS)


def check_expert_status(device=None) -> None:
    """Synchronise and raise :class:`TileCCLTimeoutError` if a wait inside a grouped product on
    ``device`` (default: the current one) gave up since the last check; the results of that call
    are undefined.  A product gives up two seconds (``TILECCL_WAIT_BUDGET_US`` if that is longer)
    and some hundred times its own running time after it began."""
    dev = torch.device("cuda" if device is None else device)
    index = torch.cuda.current_device() if dev.index is None else dev.index
    if index in _STATUS:
        torch.cuda.synchronize(index)
        words = (C.c_uint32 * _fg.STATUS_WORDS)()
        with torch.cuda.device(index):
            _native.call("tccl_expert_status", words)
        _fg.raise_on_status(torch.tensor(list(words)))


# -------------------------------------------------------------------------- routing
def _check_routing(logits, top_k, score, scale):
    _check_tensor("logits", logits, 2, tuple(_LOGIT_DTYPES))
    tokens, experts = logits.shape
    if not 1 <= experts <= MAX_ROUTED_EXPERTS:
        raise ValueError(f"logits have {experts} experts, supported are 1..{MAX_ROUTED_EXPERTS}")
    if not 1 <= top_k <= min(MAX_TOP_K, experts):
        raise ValueError(f"top_k={top_k} must be in 1..{min(MAX_TOP_K, experts)}")
    return tokens, experts, _choice("score", score, _SCORES), float(scale)


def route_experts(logits: torch.Tensor, top_k: int, *, score: str = "softmax",
                  bias: Optional[torch.Tensor] = None, groups: int = 1,
                  top_groups: Optional[int] = None, group_score: str = "top2",
                  renormalize: bool = True, scale: float = 1.0,
                  mask: Optional[torch.Tensor] = None,
                  stream: Optional[torch.cuda.Stream] = None):
    """The ``top_k`` experts of every token and their weights.

    ``logits [tokens, experts]`` (fp32, bf16 or fp16; rows may be strided) become scores
    ``p = softmax(logits)`` or ``sigmoid(logits)``.  An expert competes with ``p + bias``
    (``bias``: fp32 ``[experts]``, a balance term that does not enter the weights).  With
    ``groups > 1`` the experts form that many equal runs; a group counts by the sum of its two
    largest competing values (``group_score="max"``: by its largest) and only the
    ``top_groups`` best groups' experts stay.  Weights are ``scale * p`` of the chosen
    experts, divided by their sum if ``renormalize``.

    Returns ``(weights, ids)``: fp32 and int32 ``[tokens, top_k]``, best first, ties to the
    lower index.  The choice is exact (made in 64 bits where 32 cannot tell); weights are
    computed in 32 bits, within a few 2^-24.  A logit or bias of ``-inf`` takes an expert out; a
    token whose ``mask`` (bool ``[tokens]``) is false, or that has fewer than ``top_k`` experts
    left, gets id -1 and weight 0 in the places that stay empty.  A NaN among an unmasked row's
    logits makes the row's weights NaN (its ids stay distinct and in range).  Group counts that
    are no power of two are right but slower: every row is then decided on 64-bit keys (16384
    rows of 192 experts in 6 groups 73 us, of 256 in 8 groups 25).
    """
    tokens, experts, sig, scale = _check_routing(logits, top_k, score, scale)
    if groups < 1 or groups > 32 or experts % groups:
        raise ValueError(f"groups={groups} must be in 1..32 and divide the {experts} experts")
    top_groups = groups if top_groups is None else top_groups
    if not 1 <= top_groups <= groups:
        raise ValueError(f"top_groups={top_groups} must be in 1..{groups}")
    by_max = _choice("group_score", group_score, _GROUP_SCORES)
    if bias is not None:
        _check_tensor("bias", bias, 1, (torch.float32,), logits.device, contiguous=True)
        if bias.shape[0] != experts:
            raise ValueError(f"bias has {bias.shape[0]} entries for {experts} experts")
    if mask is not None:
        _check_tensor("mask", mask, 1, (torch.bool,), logits.device, contiguous=True)
        if mask.shape[0] != tokens:
            raise ValueError(f"mask has {mask.shape[0]} entries for {tokens} tokens")
    ld = _pitch("logits", logits)
    raw, guard = _enter(stream, logits, bias, mask)
    try:
        weights = logits.new_empty((tokens, top_k), dtype=torch.float32)
        ids = logits.new_empty((tokens, top_k), dtype=torch.int32)
        _launch("tccl_expert_route", logits.data_ptr(), ld, _ptr(bias), _ptr(mask),
                weights.data_ptr(), ids.data_ptr(), tokens, experts, top_k,
                _LOGIT_DTYPES[logits.dtype], sig, groups, top_groups, by_max,
                1 if renormalize else 0, scale, raw)
    finally:
        if guard is not None:
            guard.leave()
    return weights, ids


def route_experts_backward(grad_weights: torch.Tensor, logits: torch.Tensor, ids: torch.Tensor, *,
                           score: str = "softmax", renormalize: bool = True, scale: float = 1.0,
                           stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """Gradient of the logits from ``grad_weights`` (fp32 ``[tokens, top_k]``) and the ``ids``
    that :func:`route_experts` chose.  The choice itself has no gradient (so neither has
    ``bias``); places with id -1 contribute nothing, tokens without any id get zeros."""
    if not isinstance(ids, torch.Tensor) or ids.dim() != 2:
        raise ValueError("ids must be a 2-D tensor")
    top_k = ids.shape[1]
    tokens, experts, sig, scale = _check_routing(logits, top_k, score, scale)
    _check_tensor("ids", ids, 2, (torch.int32,), logits.device, contiguous=True)
    _check_tensor("grad_weights", grad_weights, 2, (torch.float32,), logits.device, contiguous=True)
    if tuple(ids.shape) != (tokens, top_k) or tuple(grad_weights.shape) != (tokens, top_k):
        raise ValueError(f"ids {tuple(ids.shape)} and grad_weights {tuple(grad_weights.shape)} "
                         f"must both be {(tokens, top_k)}")
    ld = _pitch("logits", logits)
    raw, guard = _enter(stream, logits, ids, grad_weights)
    try:
        grad = logits.new_empty((tokens, experts))
        _launch("tccl_expert_route_backward", grad_weights.data_ptr(), logits.data_ptr(), ld,
                ids.data_ptr(), grad.data_ptr(), tokens, experts, top_k,
                _LOGIT_DTYPES[logits.dtype], sig, 1 if renormalize else 0, scale, raw)
    finally:
        if guard is not None:
            guard.leave()
    return grad


# ------------------------------------------------------------------------- slot map
@dataclass(frozen=True)
class ExpertSlots:
    """The (token, choice) pairs of a batch in the order of their experts.

    ``offsets`` int32 ``[experts + 1]``: expert ``e`` has slots ``offsets[e]:offsets[e + 1]``;
    ``token_of_slot`` int32 ``[tokens * top_k]``, -1 behind the last slot;
    ``slot_of`` int32 ``[tokens, top_k]``, -1 for a choice without a slot.
    """

    offsets: torch.Tensor
    token_of_slot: torch.Tensor
    slot_of: torch.Tensor

    def __post_init__(self) -> None:
        o, t, s = self.offsets, self.token_of_slot, self.slot_of
        try:                                      # the usual case in few steps
            if (o.dtype is t.dtype is s.dtype is torch.int32 and o.device == t.device == s.device
                    and o.dim() == t.dim() == 1 and s.dim() == 2 and s.is_contiguous()
                    and o.is_contiguous() and t.is_contiguous()
                    and 2 <= o.shape[0] <= MAX_EXPERTS + 1 and t.shape[0] == s.numel()):
                return
        except AttributeError:
            pass
        _check_tensor("offsets", self.offsets, 1, (torch.int32,), contiguous=True)
        dev = self.offsets.device
        _check_tensor("token_of_slot", self.token_of_slot, 1, (torch.int32,), dev, contiguous=True)
        _check_tensor("slot_of", self.slot_of, 2, (torch.int32,), dev, contiguous=True)
        if not 1 <= self.num_experts <= MAX_EXPERTS:
            raise ValueError(f"offsets must have 2..{MAX_EXPERTS + 1} entries")
        if self.token_of_slot.shape[0] != self.slot_of.numel():
            raise ValueError(f"token_of_slot has {self.token_of_slot.shape[0]} entries, "
                             f"slot_of {self.slot_of.numel()}")

    @property
    def num_experts(self) -> int:
        return self.offsets.shape[0] - 1

    @property
    def tokens(self) -> int:
        return self.slot_of.shape[0]

    @property
    def top_k(self) -> int:
        return self.slot_of.shape[1]

    @property
    def capacity(self) -> int:
        """Rows of a slot-ordered matrix: ``tokens * top_k``."""
        return self.token_of_slot.shape[0]


@lru_cache(maxsize=4096)
def _slots_scratch(entries: int, experts: int) -> int:
    need = C.c_int64()
    _native.call("tccl_expert_slots_workspace", entries, experts, C.byref(need))
    return need.value


def expert_slots(ids: torch.Tensor, num_experts: int, *, first_expert: int = 0,
                 stream: Optional[torch.cuda.Stream] = None) -> ExpertSlots:
    """Slot map of ``ids`` (int32 ``[tokens, top_k]``) for the experts
    ``first_expert .. first_expert + num_experts`` that live here.  Ids outside that range
    (another rank's experts, -1) get no slot.  Pairs of one expert keep the order of their
    tokens."""
    _check_tensor("ids", ids, 2, (torch.int32,), contiguous=True)
    tokens, top_k = ids.shape
    if not 1 <= num_experts <= MAX_EXPERTS:
        raise ValueError(f"num_experts={num_experts} must be in 1..{MAX_EXPERTS}")
    if not 0 <= first_expert < 1 << 31:
        raise ValueError(f"first_expert={first_expert} must not be negative")
    if top_k < 1 or tokens * top_k >= 1 << 31:
        raise ValueError(f"ids have an unsupported shape {tuple(ids.shape)}")
    raw, guard = _enter(stream, ids)
    try:
        n = tokens * top_k
        need = _slots_scratch(n, num_experts)
        # one allocation for the three parts and the scratch
        slot_of, token_of_slot, offsets, scratch = ids.new_empty(
            2 * n + num_experts + 1 + need // 4).split((n, n, num_experts + 1, need // 4))
        slot_of = slot_of.view(tokens, top_k)
        _launch("tccl_expert_slots", ids.data_ptr(), tokens, top_k, num_experts, first_expert,
                offsets.data_ptr(), token_of_slot.data_ptr(), slot_of.data_ptr(),
                scratch.data_ptr() if need else 0, raw)
    finally:
        if guard is not None:
            guard.leave()
    slots = object.__new__(ExpertSlots)           # (its parts need no second check)
    slots.__dict__.update(offsets=offsets, token_of_slot=token_of_slot, slot_of=slot_of)
    return slots


# ----------------------------------------------------------------- grouped products
def _check_product(X, W, slots, rows, b_is_nk, epilogue):
    _choice("rows", rows, _ROWS)
    epi = _choice("epilogue", epilogue, _EPILOGUES)
    if not isinstance(slots, ExpertSlots):
        raise ValueError("slots must be an ExpertSlots")
    _check_tensor("X", X, 2, _HALF)
    _check_tensor("W", W, 3, (X.dtype,), X.device)
    if slots.offsets.device != X.device:
        raise ValueError(f"slots are on {slots.offsets.device}, X is on {X.device}")
    E = W.shape[0]
    N, K = (W.shape[1], W.shape[2]) if b_is_nk else (W.shape[2], W.shape[1])
    if E != slots.num_experts:
        raise ValueError(f"W has {E} experts, slots {slots.num_experts}")
    if X.shape[1] != K:
        raise ValueError(f"inner dimensions differ: X is {tuple(X.shape)}, W is {tuple(W.shape)}")
    want = slots.tokens if rows == "tokens" else slots.capacity
    if X.shape[0] != want:
        raise ValueError(f"X has {X.shape[0]} rows, expected {want} for rows={rows!r}")
    if K < 8 or N < 8 or K % 8 or N % 8:
        raise ValueError(f"K={K} and N={N} must be multiples of 8 (16-byte rows)")
    if epi and N % _fg.BLOCK_N:
        raise ValueError(f"epilogue 'silu_gate' needs N={N} to be a multiple of {_fg.BLOCK_N} "
                         "(128 gate columns followed by 128 up columns)")
    return E, K, N, epi


def _check_rows(name, t, shape, like, dtype=None):
    _check_tensor(name, t, 2, (dtype or like.dtype,), like.device)
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} is {tuple(t.shape)}, expected {shape}")
    return _aligned(name, t)


def _aligned(name, t) -> int:
    ld = _pitch(name, t)
    if ld % 8 or t.data_ptr() % 16:
        raise ValueError(f"{name} must have 16-byte aligned rows")
    return ld


@lru_cache(maxsize=4096)
def _scratch_sizes(device: int, slots: int, k: int) -> tuple:
    a, b = C.c_int64(), C.c_int64()
    _native.call("tccl_expert_gemm_scratch", slots, k, C.byref(a), C.byref(b))
    return a.value, b.value


_PER_THREAD_STREAM = 2                    # the handle of every thread's own default stream


def _stream_key(index: int, raw: int):
    """What tells the current stream (handle ``raw``) of a device from every other one.  PyTorch
    never destroys its own streams; the handle of another library's may be given out again while
    the stream that had it is still at work, its number is not."""
    if raw == 0 or torch.cuda.current_stream(index).stream_id != raw:
        return raw
    number = C.c_uint64()
    _native.call("tccl_stream_id", raw, C.byref(number))
    return (number.value,)


def _counters(dev, raw, nbytes):
    """(address, tensor to keep until the launch) of zeroed counters for one product."""
    capturing = torch.cuda.is_current_stream_capturing()
    arena = _ARENAS.get(dev.index)
    address = None if capturing or arena is None else arena.by_stream.get(raw)
    if address is None and raw == _PER_THREAD_STREAM and not capturing:
        address = 0
    if address is None:
        key = None if capturing else _stream_key(dev.index, raw)
        with _STATE_LOCK:
            if dev.index not in _ARENAS:
                _device_state(dev.index)
            arena = _ARENAS[dev.index]
            address = 0 if capturing else arena.by_stream.get(key, 0)
            if not address:
                address = arena.take(nbytes)
                if address and not capturing:
                    arena.by_stream[key] = address
    if address:
        return address, None
    t = torch.zeros(nbytes, dtype=torch.uint8, device=dev)          # in a capture: by the graph itself
    return t.data_ptr(), t


def _gather(X, slots, raw):
    """``X``'s rows in slot order."""
    S, K = slots.capacity, X.shape[1]
    xs = X.new_empty((S, K))
    _launch("tccl_expert_gather", X.data_ptr(), _aligned("X", X), X.shape[0],
            slots.token_of_slot.data_ptr(), xs.data_ptr(), K, S, K, raw)
    return xs


def _refuse_overlap(out, **inputs) -> None:
    """``out`` is written while the inputs are read: it may lie beside them in one buffer (other
    columns of the same rows), but not over them."""
    a0, pitch = out.data_ptr(), out.stride(0) * out.element_size()
    a1 = a0 + ((out.shape[0] - 1) * out.stride(0) + out.shape[1]) * out.element_size()
    for name, t in inputs.items():
        if t is None:
            continue
        b0, count = t.data_ptr(), t.numel()
        if count and not t.is_contiguous():
            count = sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1
        if a0 >= b0 + count * t.element_size() or b0 >= a1 or count == 0 or out.numel() == 0:
            continue
        if t.dim() == 2 and t.shape[0] > 1 and out.shape[0] > 1 and t.stride(0) * t.element_size() == pitch:
            shift = (b0 - a0) % pitch
            if shift >= out.shape[1] * out.element_size() and \
                    shift + t.shape[1] * t.element_size() <= pitch:
                continue
        raise ValueError(f"out overlaps {name}")


def _maps(slots) -> dict:
    return {"slots.offsets": slots.offsets, "slots.token_of_slot": slots.token_of_slot,
            "slots.slot_of": slots.slot_of}


def _product(X, W, slots, out, b_is_nk, epi, dh, raw, gathered=None):
    """One launch of the grouped product; every argument is checked already.  ``gathered``: scratch
    for the rows of ``X`` in slot order, when it has one row per token."""
    E = W.shape[0]
    N, K = (W.shape[1], W.shape[2]) if b_is_nk else (W.shape[2], W.shape[1])
    d = _native.ExpertGemm()
    d.dtype, d.epilogue, d.experts, d.w_nk = _fg.dtype_code(X.dtype), epi, E, 1 if b_is_nk else 0
    d.k, d.n, d.slots = K, N, slots.capacity
    d.offsets = slots.offsets.data_ptr()
    d.x, d.w, d.out, d.dh = X.data_ptr(), W.data_ptr(), out.data_ptr(), _ptr(dh)
    if gathered is not None:
        d.token_of_slot, d.x_slots = slots.token_of_slot.data_ptr(), gathered.data_ptr()
        d.x_rows = X.shape[0]
        _fg.count_launches(1)
    d.ldx, d.ldw, d.ldo = _aligned("X", X), _aligned("W", W), _aligned("out", out)
    rows_w, cols_w = W.shape[1], W.shape[2]
    d.w_expert = W.stride(0) if E > 1 else rows_w * d.ldw
    apart = d.w_expert >= (rows_w - 1) * d.ldw + cols_w
    between = d.w_expert >= cols_w and d.ldw >= (E - 1) * d.w_expert + cols_w   # [K, E, N] in memory
    if not (apart or between) or d.w_expert % 8:
        raise ValueError("W's experts overlap or are not 16-byte aligned")
    d.ld_dh = 0 if dh is None else _aligned("grad_out", dh)
    d.status, d.wait_budget_ns = _status_ptr(X.device), _wait_budget_ns()
    partial_bytes, counter_bytes = _scratch_sizes(X.device.index, d.slots, K)
    partial = None
    if partial_bytes:
        partial = torch.empty(partial_bytes, dtype=torch.uint8, device=X.device)
        d.counters, keep = _counters(X.device, raw, counter_bytes)
        d.partial = partial.data_ptr()
    _launch("tccl_expert_gemm", C.byref(d), raw)


def expert_gemm(X: torch.Tensor, W: torch.Tensor, slots: ExpertSlots,
                out: Optional[torch.Tensor] = None, *, rows: str = "tokens",
                b_is_nk: bool = False, epilogue: str = "none",
                out_dtype: Optional[torch.dtype] = None,
                stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """``out[s] = X[row of slot s] @ W[expert of slot s]`` (fp16 / bf16, fp32 accumulation).

    ``rows="tokens"``: ``X [tokens, K]``, gathered through the slot map; ``rows="slots"``: ``X
    [tokens * top_k, K]``, one row per slot.  ``W`` is ``[experts, K, N]``, or ``[experts, N,
    K]`` with ``b_is_nk``.  ``epilogue="silu_gate"`` takes every 256 columns of the product as
    128 gate columns followed by 128 up columns (``models.pack_gate_up`` of every expert) and
    writes ``silu(gate) * up``, half as wide.  Rows of ``out [tokens * top_k, N]`` behind the
    last slot keep what they held.  ``out`` must not overlap an input, the slot map included.  ``out_dtype``:
    ``X.dtype`` (default, or that of ``out``) or, without the gate, ``torch.float32``.
    ``rows="tokens"`` takes scratch memory for ``tokens * top_k`` rows of ``X``.
    """
    E, K, N, epi = _check_product(X, W, slots, rows, b_is_nk, epilogue)
    shape = (slots.capacity, N // 2 if epi else N)
    if out_dtype is None:
        out_dtype = X.dtype if out is None else out.dtype
    if out_dtype not in (X.dtype, torch.float32):
        raise TypeError(f"out_dtype must be {X.dtype} or torch.float32, got {out_dtype}")
    if out_dtype == torch.float32:
        if epi:
            raise TypeError("epilogue 'silu_gate' writes the operands' dtype")
        epi = _EPI_FLOAT
    if out is not None:
        _check_rows("out", out, shape, X, out_dtype)
        _refuse_overlap(out, X=X, W=W, **_maps(slots))
    raw, guard = _enter(stream, X, W, slots.offsets, slots.token_of_slot, out)
    try:
        if out is None:
            out = X.new_empty(shape, dtype=out_dtype)
        # Tokens' rows are put in slot order by a copy kernel first.  (8192 tokens x 2 of 4096 x
        # 28672: 2.5 ms, 8.4 with the TMA unit's four rows per copy inside the product, 6.0 with
        # copies by its threads.  Not compared for few tokens since the products became faster.)
        gathered = X.new_empty((slots.capacity, K)) if rows == "tokens" else None
        _product(X, W, slots, out, b_is_nk, epi, None, raw, gathered)
    finally:
        if guard is not None:
            guard.leave()
    return out


def expert_gemm_backward(grad_out: torch.Tensor, X: torch.Tensor, W: torch.Tensor,
                         slots: ExpertSlots, *, rows: str = "tokens", b_is_nk: bool = False,
                         epilogue: str = "none", stream: Optional[torch.cuda.Stream] = None):
    """``(grad_X, grad_W)`` of :func:`expert_gemm` for ``grad_out`` (shaped like its result).

    With ``epilogue="silu_gate"`` gate and up are computed again from ``X`` and ``W``, so the
    forward pass keeps nothing.  Their gradients are rounded to the operands' 16 bits before the two
    products that read them, half a step per element (the tensor cores take no wider operand
    beside a 16-bit one): in bf16 ``grad_X`` and ``grad_W`` are then 2.4e-3 off on the whole
    instead of 1.7e-3, and in fp16 they have to stay below 65504.

    ``grad_X`` has ``X``'s shape: with ``rows="tokens"`` the sum over a token's slots (zero for a
    token without one), with ``rows="slots"`` one row per slot, undefined behind the last slot.
    ``grad_W`` has ``W``'s shape and is contiguous; experts without a slot get zeros.
    """
    E, K, N, epi = _check_product(X, W, slots, rows, b_is_nk, epilogue)
    _check_rows("grad_out", grad_out, (slots.capacity, N // 2 if epi else N), X)
    S = slots.capacity
    raw, guard = _enter(stream, X, W, grad_out, slots.offsets, slots.token_of_slot, slots.slot_of)
    try:
        # (once in slot order for both products that read X)
        xs = _gather(X, slots, raw) if rows == "tokens" else X
        dy = grad_out
        if epi:
            # gate and up again, their gradients straight from the accumulators (one rounding
            # to 16 bits: the operand type of the two products that follow)
            dy = X.new_empty((S, N))
            _product(xs, W, slots, dy, b_is_nk, _EPI_SILU_GATE_GRAD, grad_out, raw)
        # A token's slots are summed in fp32 and rounded once: with 16-bit rows in between the
        # error grew by a quarter, the call is 3 % faster.
        grad_rows = X.new_empty((S, K), dtype=torch.float32 if rows == "tokens" else X.dtype)
        _product(dy, W, slots, grad_rows, not b_is_nk, _EPI_FLOAT if rows == "tokens" else 0, None, raw)
        grad_X = grad_rows
        if rows == "tokens":
            grad_X = X.new_empty((slots.tokens, K))
            _combine(grad_rows, K, slots, None, None, 0, grad_X, K, raw)
        grad_W = X.new_empty(W.shape)
        a, b = (dy, xs) if b_is_nk else (xs, dy)
        d = _native.ExpertWeightGrad()
        d.dtype, d.experts, d.slots = _fg.dtype_code(X.dtype), E, S
        d.offsets = slots.offsets.data_ptr()
        d.m, d.n = a.shape[1], b.shape[1]
        d.a, d.b, d.out = a.data_ptr(), b.data_ptr(), grad_W.data_ptr()
        d.lda, d.ldb = _aligned("X", a), _aligned("X", b)
        d.status, d.wait_budget_ns = _status_ptr(X.device), _wait_budget_ns()
        _launch("tccl_expert_weight_grad", C.byref(d), raw)
    finally:
        if guard is not None:
            guard.leave()
    return grad_X, grad_W


# -------------------------------------------------------------------------- combine
def _combine(H, ld_h, slots, weights, add, ld_add, out, ld_out, raw):
    tokens, top_k = slots.slot_of.shape
    _launch("tccl_expert_combine", H.data_ptr(), ld_h, slots.slot_of.data_ptr(), _ptr(weights),
            _ptr(add), ld_add, out.data_ptr(), ld_out, tokens, tokens * top_k, top_k, H.shape[1],
            _fg.dtype_code(out.dtype), 1 if H.dtype == torch.float32 else 0, raw)


def _check_combine(H, slots, weights):
    if not isinstance(slots, ExpertSlots):
        raise ValueError("slots must be an ExpertSlots")
    _check_tensor("H", H, 2, _HALF, slots.offsets.device)
    if H.shape[0] != slots.capacity:
        raise ValueError(f"H has {H.shape[0]} rows, expected {slots.capacity}")
    if H.shape[1] < 8 or H.shape[1] % 8:
        raise ValueError(f"H has {H.shape[1]} columns, which must be a multiple of 8")
    if weights is not None:
        _check_tensor("weights", weights, 2, (torch.float32,), H.device, contiguous=True)
        if weights.shape != slots.slot_of.shape:
            raise ValueError(f"weights are {tuple(weights.shape)}, expected "
                             f"{tuple(slots.slot_of.shape)}")
    return _aligned("H", H)


def expert_combine(H: torch.Tensor, slots: ExpertSlots, weights: Optional[torch.Tensor] = None,
                   out: Optional[torch.Tensor] = None, *, add: Optional[torch.Tensor] = None,
                   stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """``out[t] = add[t] + sum_j weights[t, j] * H[slot_of[t, j]]`` in fp32, rounded once.

    ``H [tokens * top_k, N]`` is slot-ordered (fp16 / bf16), ``weights`` fp32 ``[tokens,
    top_k]`` (None: all ones), ``add [tokens, N]`` a residual or a shared expert's output.
    Choices without a slot add nothing.  ``out`` may be ``add`` (in place) but must not overlap
    another input, the slot map included.
    """
    ld_h = _check_combine(H, slots, weights)
    shape = (slots.tokens, H.shape[1])
    ld_add = 0 if add is None else _check_rows("add", add, shape, H)
    ld_out = shape[1]
    if out is not None:
        ld_out = _check_rows("out", out, shape, H)
        same = add is not None and out.data_ptr() == add.data_ptr() and out.stride() == add.stride()
        _refuse_overlap(out, H=H, add=None if same else add, weights=weights, **_maps(slots))
    raw, guard = _enter(stream, H, weights, add, slots.slot_of, out)
    try:
        if out is None:
            out = H.new_empty(shape)
        _combine(H, ld_h, slots, weights, add, ld_add, out, ld_out, raw)
    finally:
        if guard is not None:
            guard.leave()
    return out


def expert_combine_backward(grad_out: torch.Tensor, H: torch.Tensor, slots: ExpertSlots,
                            weights: torch.Tensor, *,
                            stream: Optional[torch.cuda.Stream] = None):
    """``(grad_H, grad_weights)`` of :func:`expert_combine`.  Rows of ``grad_H`` behind the last
    slot are undefined; choices without a slot have weight gradient 0.  (The gradient of
    ``add`` is ``grad_out`` itself.)"""
    if weights is None:
        raise ValueError("weights must be a 2-D tensor")
    ld_h = _check_combine(H, slots, weights)
    ld_dy = _check_rows("grad_out", grad_out, (slots.tokens, H.shape[1]), H)
    raw, guard = _enter(stream, H, weights, grad_out, slots.slot_of)
    try:
        grad_H = H.new_empty(H.shape)
        grad_weights = weights.new_empty(weights.shape)
        _launch("tccl_expert_combine_backward", grad_out.data_ptr(), ld_dy, H.data_ptr(), ld_h,
                slots.slot_of.data_ptr(), weights.data_ptr(), grad_H.data_ptr(), H.shape[1],
                grad_weights.data_ptr(),
                slots.tokens, slots.capacity, slots.top_k, H.shape[1], _fg.dtype_code(H.dtype), raw)
    finally:
        if guard is not None:
            guard.leave()
    return grad_H, grad_weights
