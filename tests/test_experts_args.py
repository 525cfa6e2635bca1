"""Mixture-of-experts operators: what they refuse, checked without a GPU.

Shapes, types and ranges are checked before the device is touched, so plain CPU tensors reach
every refusal; a call that passes them all is refused for its device."""

import ctypes as C
import threading
from types import SimpleNamespace

import pytest
import torch

from tileccl_b200 import _native, ops


def _slots(tokens=4, top_k=2, experts=3):
    n = tokens * top_k
    return ops.ExpertSlots(torch.zeros(experts + 1, dtype=torch.int32),
                           torch.zeros(n, dtype=torch.int32),
                           torch.zeros(tokens, top_k, dtype=torch.int32))


@pytest.mark.parametrize("kwargs, error", [
    (dict(top_k=0), ValueError), (dict(top_k=9), ValueError), (dict(score="relu"), ValueError),
    (dict(groups=3), ValueError), (dict(groups=0), ValueError),
    (dict(groups=4, top_groups=5), ValueError), (dict(groups=4, top_groups=0), ValueError),
    (dict(groups=4, group_score="mean"), ValueError),
    (dict(bias=torch.zeros(7)), ValueError),
    (dict(bias=torch.zeros(8, dtype=torch.float16)), TypeError),
    (dict(bias=torch.zeros(16)[::2]), ValueError),
    (dict(mask=torch.ones(4)), TypeError), (dict(mask=torch.ones(3, dtype=torch.bool)), ValueError),
    (dict(), ValueError),                                        # right, but on the CPU
])
def test_route_refusals(kwargs, error):
    kwargs.setdefault("top_k", 2)
    with pytest.raises(error):
        ops.route_experts(torch.zeros(4, 8), **kwargs)


def test_route_refuses_other_layouts_and_types():
    with pytest.raises(ValueError):
        ops.route_experts(torch.zeros(8), 2)
    with pytest.raises(TypeError):
        ops.route_experts(torch.zeros(4, 8, dtype=torch.float64), 2)
    with pytest.raises(ValueError):
        ops.route_experts(torch.zeros(8, 4).t(), 2)              # unit stride along tokens
    with pytest.raises(ValueError, match="overlap"):
        ops.route_experts(torch.zeros(1, 8).expand(4, 8), 2)
    with pytest.raises(ValueError, match="experts"):
        ops.route_experts(torch.zeros(4, 513), 2)
    with pytest.raises(ValueError, match="CUDA"):
        ops.route_experts(torch.zeros(4, 8), 2)


def test_route_backward_refusals():
    logits, ids = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32)
    for g, i in [(torch.zeros(4, 3), ids), (torch.zeros(3, 2), ids),
                 (torch.zeros(4, 2), torch.zeros(5, 2, dtype=torch.int32)),
                 (torch.zeros(4, 4)[:, ::2], ids)]:
        with pytest.raises(ValueError):
            ops.route_experts_backward(g, logits, i)
    with pytest.raises(TypeError):
        ops.route_experts_backward(torch.zeros(4, 2), logits, ids.long())
    with pytest.raises(TypeError):
        ops.route_experts_backward(torch.zeros(4, 2).half(), logits, ids)


def test_slot_refusals():
    ids = torch.zeros(4, 2, dtype=torch.int32)
    for bad in (ids[0], ids[:, :0], ids.t()):
        with pytest.raises(ValueError):
            ops.expert_slots(bad, 3)
    with pytest.raises(TypeError):
        ops.expert_slots(ids.long(), 3)
    for n, first in ((0, 0), (1025, 0), (3, -1)):
        with pytest.raises(ValueError):
            ops.expert_slots(ids, n, first_expert=first)
    with pytest.raises(ValueError, match="CUDA"):
        ops.expert_slots(ids, 3)
    with pytest.raises(ValueError):
        ops.ExpertSlots(torch.zeros(4, dtype=torch.int32), torch.zeros(7, dtype=torch.int32), ids)
    with pytest.raises(TypeError):
        ops.ExpertSlots(torch.zeros(4), torch.zeros(8, dtype=torch.int32), ids)


@pytest.mark.parametrize("change, error", [
    (dict(rows="experts"), ValueError), (dict(epilogue="gelu"), ValueError),
    (dict(epilogue="silu_gate"), ValueError),                    # N is no multiple of 256
    (dict(b_is_nk=True), ValueError),                            # inner dimensions differ
    (dict(rows="slots"), ValueError),                            # 4 rows for 8 slots
    (dict(W=torch.zeros(2, 16, 24).half()), ValueError),         # experts differ
    (dict(W=torch.zeros(3, 16, 24).bfloat16()), TypeError),
    (dict(W=torch.zeros(16, 24).half()), ValueError),
    (dict(X=torch.zeros(4, 16)), TypeError),
    (dict(X=torch.zeros(4, 12).half(), W=torch.zeros(3, 12, 24).half()), ValueError),
    (dict(W=torch.zeros(3, 16, 20).half()), ValueError),
    (dict(out=torch.zeros(8, 23).half()), ValueError),
    (dict(out=torch.zeros(8, 24).double()), TypeError),
    (dict(out=torch.zeros(8, 24), out_dtype=torch.float16), TypeError),
    (dict(out_dtype=torch.bfloat16), TypeError),
    (dict(W=torch.zeros(3, 16, 256).half(), epilogue="silu_gate", out_dtype=torch.float32), TypeError),
    (dict(out=torch.zeros(8, 28).half()[:, :24]), ValueError),   # rows not 16-byte aligned
    (dict(slots=None), ValueError),
    (dict(), ValueError),                                        # right, but on the CPU
])
def test_product_refusals(change, error):
    args = dict(X=torch.zeros(4, 16).half(), W=torch.zeros(3, 16, 24).half(), slots=_slots())
    args.update(change)
    with pytest.raises(error):
        ops.expert_gemm(**args)


def test_backward_and_combine_refusals():
    s = _slots()
    X, W = torch.zeros(4, 16).half(), torch.zeros(3, 16, 24).half()
    with pytest.raises(ValueError):
        ops.expert_gemm_backward(torch.zeros(4, 24).half(), X, W, s)      # 8 slots
    with pytest.raises(TypeError):
        ops.expert_gemm_backward(torch.zeros(8, 24), X, W, s)
    H, w = torch.zeros(8, 16).half(), torch.zeros(4, 2)
    for args, kw in [((H[:4], s, w), {}), ((H, s, w[:3]), {}), ((H, s, w[:, :1]), {}),
                     ((torch.zeros(8, 12).half(), s, w), {}),
                     ((H, s, w), dict(add=torch.zeros(8, 16).half())),
                     ((H, s, w), dict(out=torch.zeros(4, 8).half())),
                     ((H, None, w), {}), ((H, s, w), {})]:
        with pytest.raises(ValueError):
            ops.expert_combine(*args, **kw)
    with pytest.raises(TypeError):
        ops.expert_combine(H.float(), s, w)
    with pytest.raises(TypeError):
        ops.expert_combine(H, s, w.half())
    with pytest.raises(ValueError):
        ops.expert_combine_backward(torch.zeros(4, 16).half(), H, s, None)
    with pytest.raises(ValueError):
        ops.expert_combine_backward(torch.zeros(8, 16).half(), H, s, w)


def test_results_may_lie_beside_their_inputs_but_not_over_them():
    s = _slots(tokens=8, top_k=1)
    big = torch.zeros(8, 64).half()
    W = torch.zeros(3, 16, 24).half()
    X, beside, over = big[:, :16], big[:, 16:40], big[:, 8:32]
    with pytest.raises(ValueError, match="CUDA"):                # right, but on the CPU
        ops.expert_gemm(X, W, s, beside)
    with pytest.raises(ValueError, match="overlaps X"):
        ops.expert_gemm(X, W, s, over)
    with pytest.raises(ValueError, match="overlaps W"):
        ops.expert_gemm(X, W, s, W.view(-1)[:8 * 24].view(8, 24))
    H, add = big[:, :16], torch.zeros(8, 16).half()
    with pytest.raises(ValueError, match="overlaps H"):
        ops.expert_combine(H, s, None, H)
    with pytest.raises(ValueError, match="CUDA"):                # in place over the residual
        ops.expert_combine(H, s, None, add, add=add)
    pair = torch.zeros(8, 24).half()
    with pytest.raises(ValueError, match="overlaps add"):
        ops.expert_combine(H, s, None, pair[:, :16], add=pair[:, 8:])


@pytest.mark.parametrize("part", ["offsets", "token_of_slot", "slot_of"])
def test_results_may_not_lie_over_the_slot_map(part):
    memory = torch.zeros(256, dtype=torch.int32)
    parts = dict(offsets=torch.zeros(4, dtype=torch.int32), token_of_slot=torch.zeros(8, dtype=torch.int32),
                 slot_of=torch.zeros(4, 2, dtype=torch.int32))
    parts[part] = memory[20:20 + parts[part].numel()].view(parts[part].shape)
    s = ops.ExpertSlots(**parts)
    over = memory.view(torch.float16)
    with pytest.raises(ValueError, match=f"overlaps slots.{part}"):
        ops.expert_gemm(torch.zeros(4, 16).half(), torch.zeros(3, 16, 24).half(), s, over[:8 * 24].view(8, 24))
    with pytest.raises(ValueError, match=f"overlaps slots.{part}"):
        ops.expert_combine(torch.zeros(8, 16).half(), s, None, over[:4 * 16].view(4, 16))
    with pytest.raises(ValueError, match="CUDA"):                # beside it
        ops.expert_gemm(torch.zeros(4, 16).half(), torch.zeros(3, 16, 24).half(), s,
                        over[64:64 + 8 * 24].view(8, 24))


def test_native_entries_check_their_arguments():
    """The C entries refuse on their own (another binding may call them)."""
    lib = _native.load()
    ok = [64, 8, 0, 0, 64, 64, 4, 8, 2, 2, 0, 1, 1, 0, 1, 1.0, 0]
    for i, v in [(0, 0), (1, 4), (6, -1), (7, 0), (7, 513), (8, 0), (8, 9), (9, 3), (11, 3),
                 (12, 2)]:
        args = list(ok)
        args[i] = v
        assert lib.tccl_expert_route(*args) == 1, (i, v)
    d = _native.ExpertGemm()
    fields = dict(dtype=0, epilogue=0, experts=3, w_nk=0, k=16, n=24, slots=8, offsets=64, x=64, w=64, out=64, dh=0, ldx=16, ldw=24, w_expert=384, ldo=24, partial=0,
                  counters=0, token_of_slot=0, x_slots=0, x_rows=0)
    for name, bad in [("dtype", 2), ("epilogue", 4), ("epilogue", 1), ("experts", 0),
                      ("experts", 1025), ("k", 12), ("n", 20), ("k", 0), ("ldx", 12), ("x", 72),
                      ("slots", -1), ("slots", 1 << 31), ("x", 0), ("offsets", 0),
                      ("partial", 64), ("token_of_slot", 64)]:
        for k, v in fields.items():
            setattr(d, k, v)
        setattr(d, name, bad)
        assert lib.tccl_expert_gemm(C.byref(d), 0) == 1, (name, bad)
    assert lib.tccl_expert_slots(64, 4, 2, 1025, 0, 64, 64, 64, 0, 0) == 1
    assert lib.tccl_expert_slots(64, 1 << 30, 2, 8, 0, 64, 64, 64, 0, 0) == 1
    assert lib.tccl_expert_slots(64, 1 << 16, 2, 8, 0, 64, 64, 64, 0, 0) == 1   # no workspace
    assert lib.tccl_expert_combine(64, 16, 64, 64, 0, 0, 64, 16, 4, 8, 2, 12, 0, 0, 0) == 1
    assert lib.tccl_expert_combine(64, 16, 64, 64, 0, 0, 64, 16, 4, 8, 2, 16, 2, 0, 0) == 1
    assert b"" != lib.tccl_last_error()


class _Rank:
    """What a block reads of a context before it allocates anything."""

    def __init__(self, rank=0, world_size=2):
        self.rank, self.world_size = rank, world_size


@pytest.mark.parametrize("change", [dict(tokens=7), dict(ffn=257), dict(ffn=384), dict(hidden=60),
                                    dict(experts=6), dict(top_k=0), dict(top_k=9)])
def test_moe_block_refusals(change):
    from tileccl_b200.models import TPMoE

    args = dict(tokens=8, hidden=64, ffn=512, experts=8, top_k=2)
    args.update(change)
    with pytest.raises(ValueError):
        TPMoE(_Rank(), **args)


# ----------------------------------------------------- state shared by host threads
def _together(call, arguments):
    """``call`` on every one of ``arguments``, each in a thread of its own."""
    results = [None] * len(arguments)

    def one(i):
        results[i] = call(*arguments[i])

    threads = [threading.Thread(target=one, args=(i,)) for i in range(len(arguments))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    return results


def _meet(barrier):
    """Waits for the other thread, unless a lock keeps it away."""
    try:
        barrier.wait(0.5)
    except threading.BrokenBarrierError:
        pass


@pytest.fixture
def shared_state(monkeypatch):
    from tileccl_b200.kernels import experts

    monkeypatch.setattr(experts, "_ARENAS", {})
    monkeypatch.setattr(experts, "_STATUS", {}, raising=False)
    monkeypatch.setattr(experts, "_stream_key", lambda index, raw: raw, raising=False)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return experts


@pytest.mark.parametrize("streams", [(1001, 1001), (1001, 1002)])
def test_first_products_of_two_threads_share_one_arena(shared_state, monkeypatch, streams):
    """Both threads find no counters yet: one arena is made and kept, so that no piece is handed out
    twice."""
    experts, made, meet = shared_state, [], threading.Barrier(2)

    class Arena(experts._CounterArena):
        def __init__(self, *args):
            made.append(self)
            _meet(meet)
            super().__init__(*args)

    def state(fn, status, counters, nbytes):
        status._obj.value, counters._obj.value, nbytes._obj.value = 64, 4096, 4096

    monkeypatch.setattr(experts, "_CounterArena", Arena)
    monkeypatch.setattr(experts._native, "call", state)
    got = _together(experts._counters, [(SimpleNamespace(index=7), raw, 128) for raw in streams])
    assert len(made) == 1 and experts._ARENAS[7] is made[0] and experts._STATUS[7] == 64
    kept = made[0].by_stream
    assert [address for address, _ in got] == [kept[raw] for raw in streams]
    assert (got[0][0] == got[1][0]) == (streams[0] == streams[1])


def test_two_threads_never_get_the_same_counters(shared_state):
    """A piece that one thread is about to take is not given to another."""
    experts, meet = shared_state, threading.Barrier(2)

    class Arena(experts._CounterArena):
        def __init__(self):
            self.address, self.BYTES, self.by_stream, self.at = 1 << 20, 4096, {}, 0

        @property
        def used(self):
            at = self.at
            _meet(meet)
            return at

        @used.setter
        def used(self, value):
            self.at = value

    experts._ARENAS[7] = Arena()
    got = _together(experts._counters, [(SimpleNamespace(index=7), raw, 128) for raw in (1001, 1002)])
    assert abs(got[0][0] - got[1][0]) >= 128


def test_status_words_come_with_the_arena(shared_state, monkeypatch):
    """Looked up once by whoever is first, and the arena that pieces were taken from stays."""
    experts, calls, meet = shared_state, [], threading.Barrier(2)

    def state(fn, status, counters, nbytes):
        calls.append(fn)
        _meet(meet)
        status._obj.value, counters._obj.value, nbytes._obj.value = 64, 4096, 4096

    monkeypatch.setattr(experts._native, "call", state)
    dev = SimpleNamespace(index=7)
    assert _together(experts._status_ptr, [(dev,)] * 2) == [64, 64]
    arena = experts._ARENAS[7]
    experts._counters(dev, 1001, 128)
    assert experts._status_ptr(dev) == 64 and experts._ARENAS[7] is arena and len(calls) == 1


def test_streams_that_share_a_handle_do_not_share_counters(shared_state, monkeypatch):
    """A handle that is given out again belongs to another stream, and the handle of the per-thread
    default stream to one stream per thread."""
    experts, numbers = shared_state, iter([41, 42, 41])
    monkeypatch.setattr(experts, "_stream_key", lambda index, raw: (next(numbers),))
    experts._ARENAS[7] = experts._CounterArena(4096, 4096)
    dev = SimpleNamespace(index=7)
    first, second, again = (experts._counters(dev, 1001, 128)[0] for _ in range(3))
    assert first == again and abs(first - second) >= 128
    zeros = torch.zeros
    monkeypatch.setattr(torch, "zeros", lambda *shape, device=None, **kw: zeros(*shape, **kw))
    (a, keep_a), (b, keep_b) = (experts._counters(dev, 2, 128) for _ in range(2))
    assert a == keep_a.data_ptr() and b == keep_b.data_ptr() and a != b
    assert experts._ARENAS[7].used == 256


def test_a_captured_first_product_reports_and_owns_its_counters(shared_state, monkeypatch):
    experts = shared_state

    def state(fn, status, counters, nbytes):
        status._obj.value, counters._obj.value, nbytes._obj.value = 64, 4096, 4096

    monkeypatch.setattr(experts._native, "call", state)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    dev = SimpleNamespace(index=7)
    assert experts._status_ptr(dev) == 64
    first, second = experts._counters(dev, 1001, 128), experts._counters(dev, 1001, 128)
    assert first[0] != second[0] and 4096 <= min(first[0], second[0]) and experts._ARENAS[7].by_stream == {}


@pytest.mark.parametrize("setting, budget", [("3000", 2_000_000_000), ("5000000", 5_000_000_000),
                                             (None, 2_000_000_000)])
def test_a_short_budget_for_peers_does_not_end_products(monkeypatch, setting, budget):
    """Products wait for no peer: what the configuration grants a peer only ever lengthens them."""
    from tileccl_b200.kernels import experts

    if setting is None:
        monkeypatch.delenv("TILECCL_WAIT_BUDGET_US", raising=False)
    else:
        monkeypatch.setenv("TILECCL_WAIT_BUDGET_US", setting)
    seen = []
    monkeypatch.setattr(experts, "_launch", lambda fn, desc, raw: seen.append(desc._obj.wait_budget_ns))
    monkeypatch.setattr(experts, "_status_ptr", lambda dev: 0)
    monkeypatch.setattr(experts, "_scratch_sizes", lambda *args: (0, 0))
    half = lambda *shape: torch.zeros(*shape, dtype=torch.float16)
    experts._product(half(4, 16), half(3, 16, 24), _slots(), half(8, 24), False, 0, None, 0)
    assert seen == [budget]
