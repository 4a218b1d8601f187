"""The compiled binding of the serving operators (``_lib/_tklab_tensors.so``, ``csrc/binding/tensors.cpp``).

Its functions take torch tensors, look at everything a kernel relies on and
launch on the current stream; they return None, having done nothing, when some
tensor is not as the kernels take it.  The operators' Python functions call
them first and only then find out what to refuse or copy, so an ordinary
call costs no Python-side checks.  There is no fallback: without the
extension every operator raises.
"""

from __future__ import annotations

import importlib.util
import sys
import sysconfig
from pathlib import Path
from types import ModuleType

import torch  # (the extension links to the libraries that this loads)

from tklab import _native

BINDING_PATH = Path(__file__).resolve().parent / "_lib" / "_tklab_tensors.so"


STAMP_MARK = "built for: "


def binding_stamp() -> str:
    """What an extension has to have been compiled for to be loaded here: torch, its C++ ABI, CUDA, Python."""
    abi = int(torch._C._GLIBCXX_USE_CXX11_ABI)
    return f"torch {torch.__version__}, cxx11 abi {abi}, cuda {torch.version.cuda}, {sysconfig.get_config_var('SOABI')}"


def stamp_of(path: Path) -> str:
    """The stamp that the build put into the extension at ``path``, without loading it."""
    _, mark, rest = path.read_bytes().partition(STAMP_MARK.encode())
    return rest.partition(b"\0")[0].decode(errors="replace") if mark else "an unknown environment"


def load() -> ModuleType:
    """Load the extension (once)."""
    name = "_tklab_tensors"
    if name not in sys.modules:
        if not BINDING_PATH.exists():
            raise RuntimeError(
                f"{BINDING_PATH.name} is not built: run `python triton-kernel-lab_b200/build_native.py` "
                "(or __graft_entry__.build()) before using the serving operators"
            )
        if stamp_of(BINDING_PATH) != binding_stamp():
            raise RuntimeError(
                f"{BINDING_PATH.name} was built for {stamp_of(BINDING_PATH)}, this is {binding_stamp()}: run "
                "`python triton-kernel-lab_b200/build_native.py`"
            )
        _native.load()
        spec = importlib.util.spec_from_file_location(name, BINDING_PATH)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        sys.modules[name] = module
    return sys.modules[name]


class _Binding:
    """The extension's functions, looked up at the first use of each."""

    def __getattr__(self, name: str) -> object:
        function = getattr(load(), name)
        setattr(self, name, function)
        return function


binding = _Binding()


def rows_in_place(x: torch.Tensor) -> bool:
    """Whether the kernels can read ``x``: contiguous 16-byte aligned rows at strides that are multiples of 8."""
    *outer, last = x.stride()
    return (
        (last == 1 or x.shape[-1] == 1)
        and x.data_ptr() % 16 == 0
        and all(n == 1 or s % 8 == 0 for n, s in zip(x.shape, outer))
    )


def rows_repeat(x: torch.Tensor) -> bool:
    """Whether some of ``x``'s rows are one in memory (an expanded tensor)."""
    return any(s == 0 and n > 1 for s, n in zip(x.stride()[:-1], x.shape))


def dense(x: torch.Tensor) -> torch.Tensor:
    """``x`` itself if the kernels can read it, else a contiguous copy (differentiable)."""
    return x if rows_in_place(x) else x.clone(memory_format=torch.contiguous_format)


def distinct(x: torch.Tensor) -> torch.Tensor:
    """:func:`dense` for what a tensor map describes: repeated rows are copied, too."""
    return dense(x.contiguous() if rows_repeat(x) else x)


def require_cache(x: torch.Tensor, name: str) -> None:
    """Refuse a cache that would have to be copied (it is written in place, or too large) or repeats rows."""
    if not rows_in_place(x) or rows_repeat(x):
        raise ValueError(f"{name} needs contiguous, 16-byte aligned rows at distinct strides that are multiples of 8")


def contiguous(x: torch.Tensor | None) -> torch.Tensor | None:
    """``x.contiguous()``, None for None."""
    return None if x is None else x.contiguous()
