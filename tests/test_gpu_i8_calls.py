"""What the Python calls of the 8-bit linear path do besides launching: errors, other threads."""
import threading
import time

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def test_out_of_memory_is_torchs_error():
    """An output that no GPU has room for (8 TB): torch.OutOfMemoryError, which callers catch to take a smaller batch,
    and the next call works."""
    import bbh

    n = 2_000_000
    q, s = torch.zeros(n, 16, dtype=torch.int8, device=DEV), torch.ones(n, device=DEV)
    with pytest.raises(torch.OutOfMemoryError, match="out of memory"):
        bbh.linear_i8(q, s, q, s)
    assert bool((bbh.linear_i8(q[:5], s[:5], q[:7], s[:7]) == 0).all())


@pytest.mark.parametrize("name", ["rmsnorm", "rmsnorm_i8", "quantize_i8", "dequantize_i8", "linear_i8"])
def test_other_threads_run_while_a_launch_waits(name):
    """A stream takes about a thousand launches; one more waits for room. 1,500 calls behind a second of work on the
    device: the thread that makes them waits most of that second in a launch, another one goes on all the time."""
    import bbh

    x = torch.ones(2, 64, dtype=torch.float16, device=DEV)
    q, s = bbh.quantize_i8(x)
    out, wide = torch.empty_like(x), torch.empty(2, 2, dtype=torch.float16, device=DEV)
    call = {"rmsnorm": lambda: bbh.rmsnorm(x, out=out), "rmsnorm_i8": lambda: bbh.rmsnorm_i8(x),
            "quantize_i8": lambda: bbh.quantize_i8(x), "dequantize_i8": lambda: bbh.dequantize_i8(q, s, out=out),
            "linear_i8": lambda: bbh.linear_i8(q, s, q, s, out=wide)}[name]
    call()
    torch.cuda.synchronize()
    times, stop = [], threading.Event()

    def tick():
        while not stop.wait(0.002):
            times.append(time.perf_counter())

    t = threading.Thread(target=tick)
    t.start()
    try:
        began = time.perf_counter()
        torch.cuda._sleep(2_000_000_000)
        longest = 0.0
        for _ in range(1500):
            a = time.perf_counter()
            call()
            longest = max(longest, time.perf_counter() - a)
        torch.cuda.synchronize()
        ended = time.perf_counter()
    finally:
        stop.set()
        t.join()
    inside = [began, *(v for v in times if began < v < ended), ended]
    gap = max(b - a for a, b in zip(inside, inside[1:]))
    assert longest > 0.5, "no launch had to wait"
    assert gap < 0.4 * longest, (gap, longest)


_FIRST_CALLS = """
import sys, threading
sys.path[:0] = [{here!r}]
import torch, bbh
sizes = [(1, 96, 64), (12, 96, 64), (20, 200, 4096), (100, 200, 1024), (64, 384, 384), (3000, 384, 64), (3000, 1536, 64)]
g = torch.Generator(device="cuda").manual_seed(3)
args = []
for m, n, k in sizes:
    x, w = (torch.randn(r, k, generator=g, device="cuda").half() for r in (m, n))
    args.append((x, w))
torch.cuda.synchronize()
start, got, errors = threading.Barrier(8), [None] * 8, []
def run(i):
    try:
        stream = torch.cuda.Stream()
        start.wait()
        with torch.cuda.stream(stream):
            got[i] = [bbh.linear_i8(*bbh.rmsnorm_i8(x), *bbh.quantize_i8(w), gelu=True) for x, w in args]
        stream.synchronize()
    except BaseException as e:
        errors.append(e)
threads = [threading.Thread(target=run, args=(i,)) for i in range(8)]
[t.start() for t in threads]
[t.join() for t in threads]
assert not errors, errors
want = [bbh.linear_i8(*bbh.rmsnorm_i8(x), *bbh.quantize_i8(w), gelu=True) for x, w in args]
assert all(torch.equal(a, b) for r in got for a, b in zip(r, want))
assert bbh.linear_i8_device_error() == 0
print("same")
"""


def test_first_calls_of_eight_threads_at_once():
    """Threads run next to one another in these calls, the very first of a process among them."""
    import os
    import subprocess
    import sys

    import bbh

    code = _FIRST_CALLS.format(here=os.path.dirname(os.path.abspath(bbh.__file__)))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "same", r.stdout + r.stderr
