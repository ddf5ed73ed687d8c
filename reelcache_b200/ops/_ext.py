"""Access to the native extension and the per-device kernel status words.

Every persistent kernel takes an int32 status word; a bounded wait that runs out writes a nonzero
code there and the kernel returns early instead of hanging. :func:`check_status` turns a nonzero
word into :class:`~reelcache_b200.errors.DeviceStatusError` (it synchronizes, so callers use it in
tests and at step boundaries, not inside hot loops).
"""

from __future__ import annotations

import threading

import torch

from .. import _native_build
from ..errors import DeviceStatusError, UnsupportedError

_status = {}
_lock = threading.Lock()

STATUS_NAMES = {
    0x101: "TMA producer wait timed out",
    0x102: "MMA issuer wait timed out",
    0x103: "epilogue wait timed out",
    0x104: "gather producer wait timed out",
    0x105: "drain wait timed out",
    0x201: "peer flag wait timed out",
    0x301: "bad kernel argument",
    0x401: "too few free pages: the page-table call was refused and changed nothing",
    0x402: "a sequence or length of a page-table call is invalid: the call was refused and changed nothing (a release "
           "skips such sequences)",
    0x403: "a page number lies outside the pool, or a length outside the block table: such keys read as zeros or not at "
           "all, writes to them were dropped",
    0x404: "a sequence has more new tokens than max_q_len, or cu_q runs backwards or past the rows of q: rows beyond have no "
           "result",
}


def ext():
    """The loaded extension module; raises UnsupportedError naming the missing library."""
    try:
        return _native_build.load()
    except ImportError as error:
        raise UnsupportedError(str(error)) from error


def available() -> bool:
    try:
        ext()
        return True
    except UnsupportedError:
        return False


def status_word(device) -> torch.Tensor:
    device = torch.device(device)
    word = _status.get(device.index)
    if word is not None:
        return word
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    with _lock:
        word = _status.get(device.index)
        if word is None:
            word = torch.zeros(4, dtype=torch.int32, device=device)
            _status[device.index] = word
    return word


def check_status(device) -> None:
    """Raise DeviceStatusError if any kernel on ``device`` recorded a failure (synchronizes)."""
    word = status_word(device)
    codes = [code for code in word[:2].tolist() if code]  # the second word is the paged-cache operators'
    if codes:
        word.zero_()
        raise DeviceStatusError("; ".join(f"kernel status 0x{code:x}: {STATUS_NAMES.get(code, 'unknown failure')}" for code in codes))


def require_cuda(tensor: torch.Tensor, what: str) -> None:
    if tensor.device.type != "cuda":
        raise UnsupportedError(f"{what} needs CUDA tensors")
