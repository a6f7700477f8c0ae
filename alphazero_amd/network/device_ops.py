"""What the training operators (layer_norm.py, adamw.py) share: element types, streams and errors of the C ABI."""
import torch

from .. import _lib
from ..engine import EngineError

TYPE_IDS = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}   # AZ_TYPE_* of include/az_engine.h

_library = None


def library():
    """The HIP library, for calls that take a stream of PyTorch's."""
    global _library
    if _library is None:
        L = _lib.lib()
        # A stream belongs to the HIP runtime that made it.  _lib.lib() loads PyTorch's runtime first and the library then
        # uses the same one; a process that loaded the library by itself before that has two.
        with open("/proc/self/maps") as fh:
            runtimes = {line.split()[-1] for line in fh if "/libamdhip64.so" in line}
        if len(runtimes) > 1:
            raise RuntimeError("two HIP runtimes are loaded (%s): import torch before libazamd.so is loaded" % ", ".join(sorted(runtimes)))
        _library = L
    return _library


def current_stream(device_index):
    """Handle of PyTorch's current stream on a device."""
    return torch._C._cuda_getCurrentRawStream(device_index)


def check(rc):
    if rc < 0:
        raise EngineError(rc, _lib.lib().az_last_error(None).decode())


def dense(t):
    """Whether t's elements fill a run of memory without gaps and without one element standing for two."""
    if t.is_contiguous():
        return True
    want = 1
    for stride, size in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n != 1):
        if stride != want:
            return False
        want *= size
    return True


def in_memory_order(t):
    """The elements of a dense tensor as they lie in memory, one axis."""
    return t.view(-1) if t.is_contiguous() else t.as_strided((t.numel(),), (1,))
