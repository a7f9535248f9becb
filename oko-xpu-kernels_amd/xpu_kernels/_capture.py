"""Is the current stream being captured into a HIP graph?

The counterpart of the reference's ``python/xpu_kernels/_capture.py:15-34``:
kernels that would materialise a full-precision copy of a weight refuse to run
inside a capture, because a captured copy is re-made on every replay.
"""

import torch


def is_capturing() -> bool:
    try:
        return bool(torch.cuda.is_available() and torch.cuda.is_current_stream_capturing())
    except Exception:  # noqa: BLE001 - no device runtime means no capture
        return False


def refuse_default_stream_leaf() -> None:
    """Raise if the current stream is being captured.  Called for a tensor whose gradient goes
    to a graph of the default stream: the backward pass would make that stream wait for the
    capturing one, which no capture allows and which ends the process.  (A stream that can be
    captured joins the capture and is joined to it again.)"""
    if is_capturing():
        raise RuntimeError(
            "a tensor that needs a gradient is part of a graph that was made on the default stream "
            "and is still alive; its backward pass cannot be captured. Delete what holds that graph "
            "(a loss, an output) before capturing, or make it on a stream of its own")
