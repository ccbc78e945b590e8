"""Loads libisa_block_hip.so (include/isa_block.h, include/isa_train.h) and torch's binding to it, `_binding.so`.

They are the only compute path: importing fails loudly when one is missing or was built for
another ABI. torch is imported first, so that both use the HIP runtime that it loaded.
"""

from __future__ import annotations

from pathlib import Path

import torch  # noqa: F401  (loads the HIP runtime that the library must share)

from isa.kernels.transformer_ffn._hip import HipExtensionError

LIB_PATH = Path(__file__).resolve().parent / "libisa_block_hip.so"


def load():
    """The binding, checked against the library it runs."""
    try:
        from isa.kernels.transformer_block import _binding
    except ImportError as e:
        raise HipExtensionError(f"{LIB_PATH.name} or its binding cannot be loaded from {LIB_PATH.parent} ({e}); build "
                                "them with `python isa-_amd/csrc/build.py` (or __graft_entry__.build())") from e
    has = (_binding.abi_version(), _binding.train_abi_version())
    expects = (_binding.ABI_VERSION, _binding.TRAIN_ABI_VERSION)
    if has != expects:
        raise HipExtensionError(f"{LIB_PATH} has ABI versions {has}, its binding expects {expects}; rebuild them")
    return _binding
