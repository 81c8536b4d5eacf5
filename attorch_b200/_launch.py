"""
What a launch needs from the host besides its arguments, at the least cost: small calls are bound by the host, and the
public forms of these three took 6 of the 28 microseconds of a one-token call.
"""

import contextlib
import threading
from typing import Optional

import torch
from torch.autograd import forward_ad

from .linear_layer import _status_made, _status_words

_CURRENT = contextlib.nullcontext()
_making = threading.Lock()


def on(device: torch.device):
    """Context in which ``device`` is current; nothing where it is already."""
    return _CURRENT if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def stream_of(device: torch.device) -> int:
    """The current stream of ``device`` as an address."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def recorded(*tensors: Optional[torch.Tensor]) -> bool:
    """
    Whether a call goes through its autograd function: something asks for a gradient, or an input may carry a forward-mode
    tangent, which PyTorch then refuses (there are no such derivatives) where the bare call would drop it.
    """
    if forward_ad._current_level >= 0:
        return True
    return torch.is_grad_enabled() and any(tensor is not None and tensor.requires_grad for tensor in tensors)


def has_tangent(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether one of the tensors carries a forward-mode tangent."""
    return forward_ad._current_level >= 0 and \
        any(tensor is not None and forward_ad.unpack_dual(tensor).tangent is not None for tensor in tensors)


def status_of(device: torch.device) -> int:
    """
    Address of the device's status word (see ``check_status``).  All streams share it: it is written by a wait that ran out
    and by nothing else.  It is never dropped, because captured graphs hold its address.
    """
    word = _status_words.get(device.index)
    return (_new_status_word(device) if word is None else word).data_ptr()


def _new_status_word(device: torch.device) -> torch.Tensor:
    with _making:
        if device.index in _status_words:                        # another thread was first
            return _status_words[device.index]
        word = torch.empty(1, dtype=torch.int32, device=device)
        # Recorded in a capture, the zeroing would only run with the graph's replays, and ``check_status`` before the first
        # of them would read whatever is there: it runs now, on a stream that is not captured.
        capturing = torch.cuda.is_current_stream_capturing()
        stream = torch.cuda.Stream(device) if capturing else torch.cuda.current_stream(device)
        with torch.cuda.stream(stream):
            word.zero_()
        _status_made[device.index] = torch.cuda.Event()
        _status_made[device.index].record(stream)
        _status_words[device.index] = word
    return word
