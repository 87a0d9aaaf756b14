"""The int8 calls' error word of the device: waits given up by calls of other
threads, other streams and captured graphs are seen by workspace_error, and a
reset makes every thread's buffers zero again."""
import ctypes
import subprocess
import sys
import threading

import pytest
import torch

from conftest import PKG_ROOT
from gsp import _native
from gsp import int8_head as I
from gsp import triton_runtime as tr


def test_refusal():
    assert _native.load().gsp_int8_error(None, None, None) == _native.GSP_ERR_INVALID_ARGUMENT


def test_reset_replaces_every_threads_buffers(monkeypatch):
    """On the host: the buffers of two threads hold what a failed call left;
    after one thread's reset both get zeros, once, and keep their sizes."""
    cpu = torch.device("cpu", 0)
    monkeypatch.setattr(_native, "_workspace_bytes", lambda batch, vocab: 4096)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: type("S", (), {"cuda_stream": 7})())
    cleared = []
    monkeypatch.setattr(_native, "_int8_error", lambda index, set_to=None: cleared.append((index, set_to)) or 0)
    monkeypatch.setattr(_native, "_thread", threading.local())
    monkeypatch.setattr(_native, "_int8_resets", {})
    ready, reset, words = threading.Barrier(3), threading.Barrier(3), []

    def get():
        return _native._int8_buffers(cpu, 7, 1, 1, 100)[0]

    def work():
        ws = get()
        ws[4:8].view(torch.int32).fill_(1)  # as a kernel of this thread leaves it
        assert get() is ws
        ready.wait(60)
        reset.wait(60)
        fresh = get()
        words.append((int(fresh.count_nonzero()), fresh.numel() == ws.numel(), get() is fresh))

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    ready.wait(60)
    _native.reset_workspace(cpu)
    reset.wait(60)
    for t in threads:
        t.join()
    assert words == [(0, True, True)] * 2 and cleared == [(0, 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("route", tr.ROUTES)
def test_word_is_seen_everywhere_and_outlives_replays(cuda_device, route):
    """A word left by some call (here stored by hand: no wait is made to run
    out) is reported on every stream and thread, and replays of a captured
    call, whose workspace the graph zeroes, leave it; calls on several threads
    and replays by themselves report none."""
    dev = cuda_device
    vocab, hidden, batch = 5000, 256, 6
    g = torch.Generator(device=dev).manual_seed(3)
    weight = I.QuantizedRows(torch.randint(-127, 128, (vocab, hidden), generator=g, device=dev, dtype=torch.int8),
                             torch.rand(vocab, generator=g, device=dev))
    h = torch.randn(batch, hidden, generator=g, device=dev).half()
    mask = torch.randint(-2 ** 31, 2 ** 31 - 1, (batch, (vocab + 31) // 32), generator=g, device=dev, dtype=torch.int32)
    want = I.int8_grammar_logits(h, weight, mask, route=route)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = I.int8_grammar_logits(h, weight, mask, route=route)
    found = []

    def work(stream):
        with torch.cuda.stream(stream):
            stream.wait_stream(torch.cuda.default_stream(dev))
            got = I.int8_grammar_logits(h, weight, mask, route=route)
            stream.synchronize()
            found.append((_native.workspace_error(dev), all(torch.equal(a, b) for a, b in zip(got, want))))

    def threads():
        found.clear()
        torch.cuda.synchronize()
        running = [threading.Thread(target=work, args=(torch.cuda.Stream(dev),)) for _ in range(2)]
        for t in running:
            t.start()
        for t in running:
            t.join()
        return list(found)

    assert threads() == [(0, True)] * 2
    graph.replay()
    assert _native.workspace_error(dev) == 0 and all(torch.equal(a, b) for a, b in zip(out, want))
    assert _native._int8_error(0, set_to=4) == 0
    graph.replay()
    assert _native.workspace_error(dev) == 4
    assert threads() == [(4, True)] * 2
    _native.reset_workspace(dev)
    graph.replay()
    assert _native.workspace_error(dev) == 0 and threads() == [(0, True)] * 2


FIRST_CALL = """
import sys
sys.path.insert(0, sys.argv[1])
import torch
from gsp import _native, int8_head as I
dev = torch.device("cuda", 0)
h, values = torch.ones(3, 64, device=dev).half(), torch.ones(500, 64, dtype=torch.int8, device=dev)
weight = I.QuantizedRows(values, torch.ones(500, device=dev))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    logits, value, token = I.int8_grammar_logits(h, weight, None)
graph.replay()
torch.cuda.synchronize()
assert (logits == 64).all() and token.tolist() == [0, 0, 0] and _native.workspace_error(dev) == 0
print("captured first")
"""


@pytest.mark.gpu
def test_first_call_of_a_process_may_be_captured(cuda_device):
    done = subprocess.run([sys.executable, "-c", FIRST_CALL, PKG_ROOT], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "captured first" in done.stdout, done.stdout + done.stderr
