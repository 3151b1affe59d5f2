"""Linear attention and cache pages called from two host threads at once, each on a stream of its own: calls of one kernel
that need different amounts of shared memory."""
import threading

import pytest
import torch

import viby_model_b200 as V
from linear_cases import decays, make

pytestmark = pytest.mark.gpu
DEV = "cuda"


def in_two_threads(calls, rounds):
    """Runs each of two calls `rounds` times, at the same time, and returns what the last ones gave."""
    got, failed = [None, None], []
    gate = threading.Barrier(2)

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()) as _:
                gate.wait()
                for _ in range(rounds):
                    got[i] = calls[i]()
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001  (reported by the test)
            failed.append((i, repr(e)))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    torch.cuda.synchronize()
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    return got


def test_page_tables_of_few_and_of_many_pages():
    few, many = torch.randn(64, 8, device=DEV), torch.randn(8192, 8, device=DEV)
    turn = [torch.arange(n - 1, -1, -1, device=DEV) for n in (64, 8192)]
    want = [few.clone(), many.clone()]
    tables = [V.PageTable([few]), V.PageTable([many])]
    rounds = 2000  # an even number of reversals leaves every page where it was
    in_two_threads([lambda: tables[0].reorder(turn[0]), lambda: tables[1].reorder(turn[1])], rounds)
    assert torch.equal(few, want[0]) and torch.equal(many, want[1])


@pytest.mark.parametrize("segments", [1, 2])
def test_linear_attention_of_small_and_of_large_heads(segments):
    cases = [make(1, 96, 2, 2, 2, d, d, torch.float32)[:3] for d in (16, 256)]
    g = decays(2).to(DEV)
    args = [[x.to(DEV) for x in c] for c in cases]
    calls = [lambda a=a: V.linear_attention_fn(*a, g, segments=segments) for a in args]
    want = [c() for c in calls]
    for o, w in zip(in_two_threads(calls, 1500), want):
        assert torch.equal(o, w)


def first_call_of_a_thread(call):
    got = []

    def work():
        try:
            got.append(call())
        except Exception as e:  # noqa: BLE001  (reported by the test)
            got.append(e)

    torch.cuda.synchronize()
    t = threading.Thread(target=work)
    t.start()
    t.join()
    if isinstance(got[0], Exception):
        raise got[0]
    return got[0]


@pytest.mark.parametrize("kernel", ["tc", "mma", "simt"])
def test_the_first_cuda_call_of_a_host_thread(kernel):
    """No context is bound to a new thread yet, and memory comes from the allocator's cache: the call has to bind it."""
    q, k, v, do, s0, ds = (x.to(DEV) for x in make(1, 300, 2, 2, 2, 64, 64, torch.bfloat16))
    g = decays(2).to(DEV)
    calls = [lambda: V.linear_attention_fn(q, k, v, g, None, s0, True, kernel=kernel),
             lambda: V.linear_attention_bwd(q, k, v, g, do, None, s0, ds, kernel=kernel),
             lambda: (V.linear_attention_update(q[:, 0], k[:, 0], v[:, 0], s0.clone(), g),)]
    for call in calls:
        want = call()
        for a, b in zip(first_call_of_a_thread(call), want):
            assert torch.equal(a, b)


def test_the_first_convolution_of_a_host_thread():
    x, w = torch.randn(4, 512, 1152, device=DEV).bfloat16().transpose(1, 2), torch.randn(1152, 4, device=DEV).bfloat16()
    for call in (lambda: (V.causal_conv1d_fn(x, w, None, activation="silu", kernel="tma"),), lambda: V.causal_conv1d_bwd(x, w, None, x, "silu")[:1]):
        want = call()
        for a, b in zip(first_call_of_a_thread(call), want):
            assert torch.equal(a, b)
