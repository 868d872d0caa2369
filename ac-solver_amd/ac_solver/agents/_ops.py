"""The torch binding of libacx's operators on activations (csrc/binding/acx_torch.cpp -> lib/acx_torch.so): checks of arguments, outputs, scratch
memory and autograd nodes in C++, the kernels behind include/acx.h.  The library that ac_solver._acx loaded is handed to it function by
function, so there is one in the process."""
import ctypes as C
import importlib.machinery
import importlib.util
import os

import torch  # noqa: F401  (acx_torch.so binds to the libraries that this import loads)

from ac_solver import _acx

LIB_PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__)))), "lib", "acx_torch.so")
if not os.path.exists(LIB_PATH):
    raise ImportError(f"{LIB_PATH} not found: build it first (python __graft_entry__.py, or make -C ac-solver_amd/csrc)")


def _load():
    loader = importlib.machinery.ExtensionFileLoader("acx_torch", LIB_PATH)
    module = importlib.util.module_from_spec(importlib.util.spec_from_file_location("acx_torch", LIB_PATH, loader=loader))
    loader.exec_module(module)
    names = [n for n in _acx.SIGNATURES if n.startswith(("acx_scan_", "acx_block_", "acx_act8_"))] + ["acx_last_error"]
    module.bind({n: C.cast(getattr(_acx.lib, n), C.c_void_p).value for n in names}, _acx.AcxError)
    return module


ops = _load()
DTYPES = (torch.float32, torch.bfloat16, torch.float16)  # of activations
