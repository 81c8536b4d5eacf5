"""
What a launch needs from the host besides its arguments, at the least cost: small calls are bound by the host, and the
public forms of these three took 6 of the 28 microseconds of a one-token call.
"""

import contextlib

import torch

from .linear_layer import _scratch, _stream_scratch

_CURRENT = contextlib.nullcontext()


def on(device: torch.device):
    """Context in which ``device`` is current; nothing where it is already."""
    return _CURRENT if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def stream_of(device: torch.device) -> int:
    """The current stream of ``device`` as an address."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def status_of(device: torch.device, stream: int) -> int:
    """Address of the status word of a stream of ``device``, which is current (see ``check_status``)."""
    entry = _scratch.get((device.index, stream))
    if entry is None:
        if torch.cuda.is_current_stream_capturing():
            # Made inside the capture the word would be zeroed by the graph's replays only, and ``check_status`` before the
            # first of them would read whatever is there.  Any other stream's word of the device serves: it is written
            # by a wait that ran out and by nothing else.
            for (index, _), other in _scratch.items():
                if index == device.index:
                    return other['status'].data_ptr()
        entry = _stream_scratch(device)
    return entry['status'].data_ptr()
