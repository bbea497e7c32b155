"""Shared pages and shared-prefix decode called from several threads."""

from __future__ import annotations

import threading

import pytest
import torch

from tests.test_shared_prefix_gpu import DEV, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import flashattntile_b200  # noqa: F401


class _Library:
    """The library, with one function that stands in for its own."""

    def __init__(self, lib, name, function):
        self._lib, self._name, self._function = lib, name, function

    def __getattr__(self, name):
        return self._function if name == self._name else getattr(self._lib, name)


def _in_turn(monkeypatch, name, read, first, second):
    """What the library reads in a call of one thread, while another thread's call comes and
    goes between the call and the reading.  (None: that call waited for this one to end.)"""
    from flashattntile_b200 import _lib

    inside, over, got = threading.Event(), threading.Event(), {}

    def function(address, *args):
        me = threading.current_thread().name
        if me == "first":
            inside.set()
            over.wait(2.0)
        got[me] = read(address)
        return 0

    lib = _lib.load()
    monkeypatch.setattr(_lib, "load", lambda: _Library(lib, name, function))
    errors = []

    def run(call):
        try:
            call()
        except BaseException as error:  # noqa: BLE001
            errors.append(error)

    a = threading.Thread(target=run, args=(first,), name="first")
    a.start()
    assert inside.wait(20.0)

    def other():
        run(second)
        over.set()

    b = threading.Thread(target=other, name="second")
    b.start()
    a.join(), b.join()
    assert not errors
    return got


def test_a_decode_launches_with_its_own_pointers(monkeypatch):
    from flashattntile_b200 import _lib, find_shared_prefix, shared_prefix_decode_attention, value_checks

    q, cache, _ = make("f16", [3], [64], [1, 2, 3], 8, 2, 64, 16)
    q2 = q.clone()
    shared = find_shared_prefix(cache, [3])
    with value_checks(False):
        shared_prefix_decode_attention(q, cache, shared)  # kept for calls of this layout
        got = _in_turn(monkeypatch, "fat_shared_prefix_decode",
                       lambda at: _lib.SharedPrefixCall.from_address(at).decode.q,
                       lambda: shared_prefix_decode_attention(q, cache, shared),
                       lambda: [shared_prefix_decode_attention(q2, cache, shared) for _ in range(2)])
    assert got == {"first": q.data_ptr(), "second": q2.data_ptr()}


def test_a_kept_struct_is_its_threads(monkeypatch):
    """Also where both threads have called before."""
    from flashattntile_b200 import _lib, find_shared_prefix, shared_prefix_decode_attention, value_checks

    q, cache, _ = make("f16", [3], [64], [1, 2, 3], 8, 2, 64, 16)
    q2 = q.clone()
    shared = find_shared_prefix(cache, [3])
    lib, calls = _lib.load(), []

    def function(address):
        calls.append(_lib.SharedPrefixCall.from_address(address).decode.q)
        return 0

    with value_checks(False):
        monkeypatch.setattr(_lib, "load", lambda: _Library(lib, "fat_shared_prefix_decode", function))
        for _ in range(3):
            for x in (q, q2):
                t = threading.Thread(target=lambda x=x: [shared_prefix_decode_attention(x, cache, shared) for _ in range(2)])
                t.start()
                t.join()
                assert shared._packed.thread != threading.get_ident()
    assert calls == [q.data_ptr()] * 2 + [q2.data_ptr()] * 2 + ([q.data_ptr()] * 2 + [q2.data_ptr()] * 2) * 2


def test_a_page_operation_launches_with_its_own_words(monkeypatch):
    """The struct of a pool holds the stream and the error word of one call at a time."""
    from flashattntile_b200 import PagePool, _lib, value_checks

    pool = PagePool.allocate(8, 2, 32, 1, 8, 4, device=DEV)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()

    def reserve(stream):
        with torch.cuda.stream(stream):
            pool.reserve(1)

    with value_checks(False):
        got = _in_turn(monkeypatch, "fat_reserve_tokens", lambda at: _lib.PagePoolCall.from_address(at).stream,
                       lambda: reserve(a), lambda: reserve(b))
    assert got == {"first": a.cuda_stream, "second": b.cuda_stream}


@pytest.mark.parametrize("same", [True, False])
def test_two_threads_on_one_stream(same):
    """The two kernels of a call follow each other on the stream: neither thread's join
    meets the other's partials.  With one SharedPrefix and with one each."""
    from flashattntile_b200 import find_shared_prefix, shared_prefix_decode_attention, value_checks

    problems = []
    for seed in range(2):
        q, cache, _ = make("f16", [20], [320], [1 + i % 5 for i in range(20)], 8, 2, 64, 16, seed=seed)
        problems.append([q, cache, find_shared_prefix(cache, [20])])
    if same:
        problems[1][1:] = problems[0][1:]
    with value_checks(False):
        want = [shared_prefix_decode_attention(*p) for p in problems]
        torch.cuda.synchronize()
        outs, start = [[], []], threading.Barrier(2)

        def run(i):
            start.wait()
            for _ in range(400):
                outs[i].append(shared_prefix_decode_attention(*problems[i]))

        threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
        [t.start() for t in threads]
        [t.join() for t in threads]
        torch.cuda.synchronize()
    for i in range(2):
        assert len(outs[i]) == 400 and all(torch.equal(x, want[i]) for x in outs[i])
