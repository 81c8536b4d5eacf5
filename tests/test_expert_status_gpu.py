"""The status word of the experts' and 8-bit products: one a device, held for good, read by check_status."""

import pytest
import torch

import attorch_b200 as attorch
from attorch_b200 import _lib, linear_layer
from attorch_b200._launch import status_of

pytestmark = pytest.mark.gpu


def captured_call():
    """A graph of one grouped product, captured on a stream of its own, and the address its kernel reports to."""
    x, w = torch.ones(20, 32, device='cuda'), torch.ones(2, 32, 48, device='cuda')
    offsets = torch.tensor([0, 7, 20], dtype=torch.int32, device='cuda')
    attorch.grouped_linear(x, offsets, w)                     # loads the kernels outside the capture
    torch.cuda.synchronize()
    return x, w, offsets


def test_word_outlives_idle_streams_and_is_read():
    """A graph keeps the address after its stream has long been idle; what a replay stores there is reported."""
    x, w, offsets = captured_call()
    device = x.device
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        y = attorch.grouped_linear(x, offsets, w)
        address = status_of(device)
    layer = attorch.Linear(64, 64)
    rows = torch.randn(32, 64, device='cuda')
    for stream in [torch.cuda.Stream() for _ in range(linear_layer._MAX_SCRATCH_ENTRIES + 8)]:
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            layer(rows)
    attorch.check_status()                                    # drops the scratch of idle streams
    word = linear_layer._status_words[device.index]
    assert word.data_ptr() == address == status_of(device)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, torch.full_like(y, 32.0))
    word.fill_(2)                                             # what a wait that ran out stores
    with pytest.raises(_lib.LibraryError, match='device status 2'):
        attorch.check_status(device)
    attorch.check_status()


def test_word_made_inside_a_capture_is_valid_at_once():
    """No call before the capture had made a word: it is zero before the graph has run, and replays leave it alone."""
    x, w, offsets = captured_call()
    index = x.device.index
    held = linear_layer._status_words.pop(index)
    filler = torch.full((1 << 20,), -1, dtype=torch.int32, device='cuda')
    del filler                                                # memory handed out next is not zero
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
            y = attorch.grouped_linear(x, offsets, w)
        attorch.check_status()
        linear_layer._status_words[index].fill_(3)
        graph.replay()
        with pytest.raises(_lib.LibraryError, match='device status 3'):
            attorch.check_status()
        attorch.check_status()
        assert torch.equal(y, torch.full_like(y, 32.0))
    finally:
        linear_layer._status_words[index] = held


def test_check_does_not_disturb_a_capture_of_another_thread():
    """
    check_status reads on the current stream and waits for no stream that is being captured.  (In the capture mode that lets
    other threads synchronise at all: the default one is ended by any read of a device value.)
    """
    import threading
    x, w, offsets = captured_call()
    errors = []

    def check():
        try:
            attorch.check_status()
        except Exception as error:
            errors.append(error)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream(), capture_error_mode='thread_local'):
        y = attorch.grouped_linear(x, offsets, w)
        thread = threading.Thread(target=check)
        thread.start()
        thread.join()
        z = attorch.grouped_linear(x, offsets, w)
    assert not errors
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, torch.full_like(y, 32.0)) and torch.equal(y, z)


def test_threads_that_come_first_together_share_one_word():
    import threading
    x, w, offsets = captured_call()
    index = x.device.index
    held = linear_layer._status_words.pop(index)
    seen, start = [], threading.Barrier(8)

    def call():
        start.wait()
        attorch.grouped_linear(x, offsets, w)
        seen.append(status_of(x.device))

    try:
        threads = [threading.Thread(target=call) for _ in range(8)]
        for thread in threads:
            thread.start()
        for thread in threads:
            thread.join()
        assert len(seen) == 8 and set(seen) == {linear_layer._status_words[index].data_ptr()}
        attorch.check_status()
    finally:
        linear_layer._status_words[index] = held
