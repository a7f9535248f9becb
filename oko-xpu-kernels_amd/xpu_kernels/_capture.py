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


def _is_captured(stream) -> bool:
    with torch.cuda.stream(stream):
        return is_capturing()


def refuse_foreign_leaf(stream_id: int, device_index: int, device_type: int) -> None:
    """Raise if the current stream is being captured and the given one, to which the gradient
    of a leaf belongs, is not: the backward pass would make it wait for the capturing stream,
    which breaks the capture and ends the process."""
    if not is_capturing():
        return
    # (the default stream, id 0, is never captured, and asking it disturbs a capture)
    if stream_id != 0 and _is_captured(torch.cuda.Stream(
            stream_id=stream_id, device_index=device_index, device_type=device_type)):
        return
    raise RuntimeError(
        "a leaf that needs a gradient has one of a graph that was made on a stream outside of this "
        "capture and is still alive; its backward pass cannot be captured. Delete what holds that "
        "graph (a loss, an output) before capturing, or make it on the capturing stream")
