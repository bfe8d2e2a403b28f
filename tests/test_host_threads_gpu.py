"""Host threads, each with a stream of its own, call the same kernels with sizes that need different amounts of shared memory: every call
launches, whatever another thread has set in between, and the results are those of one thread."""
import threading

import pytest
import torch

import acrotensor_b200 as ab
from acrotensor_b200 import _lib
from acrotensor_b200._lib import lib

pytestmark = pytest.mark.gpu

ROUNDS, THREADS = 6000, 4            # threads of each call


def at_once(*makers):
    """Each maker's call over and over in THREADS threads, on arrays of each thread's own."""
    calls = [make() for make in makers for _ in range(THREADS)]
    streams = [torch.cuda.Stream() for _ in calls]
    expect = [[x.clone() for x in call(torch.cuda.current_stream().cuda_stream)] for call in calls]
    torch.cuda.synchronize()
    start, faults, got = threading.Barrier(len(calls)), [], [None] * len(calls)

    def work(i):
        try:
            start.wait(60)
            for n in range(ROUNDS):
                got[i] = calls[i](streams[i].cuda_stream)
                if n % 100 == 99:
                    streams[i].synchronize()
        except Exception as e:
            faults.append((i, e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not faults, faults
    assert lib().acro_b200_device_status() == _lib.OK
    for a, b in zip(expect, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def attention(d):
    """Heads of d columns of one token: the pass on the ordinary cores, whose shared memory grows with d."""
    torch.manual_seed(d)
    q, k, v = (torch.randn(1, 1, 1, d, device="cuda") for _ in range(3))
    g, state, out = torch.zeros(1, device="cuda"), torch.randn(1, 1, d, d, device="cuda"), torch.empty(1, 1, 1, d, device="cuda")

    def call(stream):
        ab.linear_attention(out, q, k, v, g, initial_state=state, stream=stream)
        return (out,)
    return call


def norm_gradient(width):
    torch.manual_seed(width)
    x, dy = torch.randn(64, width, device="cuda"), torch.randn(64, width, device="cuda")
    mean, rstd, dx = torch.zeros(64, device="cuda"), torch.ones(64, device="cuda"), torch.empty_like(x)
    dw, db = torch.empty(width, device="cuda"), torch.empty(width, device="cuda")
    scratch = torch.empty(ab.layer_norm_backward_scratch_bytes(x), dtype=torch.uint8, device="cuda")

    def call(stream):
        ab.layer_norm_backward(dx, dw, db, dy, x, mean, rstd, scratch=scratch, stream=stream)
        return dx, dw, db
    return call


def test_heads_of_different_sizes():
    at_once(lambda: attention(256), lambda: attention(72))


def test_rows_of_different_widths():
    """Groups of threads that are added up in shared memory beside rows of one group, which take none."""
    at_once(lambda: norm_gradient(100), lambda: norm_gradient(2000))


def matvec(n):
    torch.manual_seed(n)
    a, x, y = (torch.randn(64, *s, dtype=torch.float64, device="cuda") for s in ((n, n), (n,), (n,)))

    def call(stream):
        _lib.check(lib().acro_b200_batched_gemm(a.data_ptr(), x.data_ptr(), y.data_ptr(), 64, n, 1, n, _lib.OP_ASSIGN, stream))
        return (y,)
    return call


def test_contractions_of_different_sizes():
    at_once(lambda: matvec(64), lambda: matvec(8))
