"""What the training operators (layer_norm.py, adamw.py) share: the native calls behind them and the layout of tensors."""
import importlib

import torch

from .. import _lib
from ..engine import EngineError

TYPES = (torch.float32, torch.bfloat16, torch.float16)   # AZ_TYPE_* of include/az_engine.h

_binding = None


def binding():
    """csrc/az_torch.cpp: the training operators of the C ABI as PyTorch calls."""
    global _binding
    if _binding is None:
        _lib.lib()
        # A stream belongs to the HIP runtime that made it.  _lib.lib() loads PyTorch's runtime first and the library then
        # uses the same one; a process that loaded the library by itself before that has two.
        with open("/proc/self/maps") as fh:
            runtimes = {line.split()[-1] for line in fh if "/libamdhip64.so" in line}
        if len(runtimes) > 1:
            raise RuntimeError("two HIP runtimes are loaded (%s): import torch before libazamd.so is loaded" % ", ".join(sorted(runtimes)))
        try:
            _binding = importlib.import_module("._train_ops", __package__)
        except ImportError as e:
            raise ImportError("alphazero_amd: network/_train_ops.so is missing or does not load (%s) - build it with "
                              "`python -c 'import __graft_entry__ as g; g.build()'` or `make -C alphazero_amd/csrc`" % e) from e
    return _binding


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
