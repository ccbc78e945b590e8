"""Registers of the built library's kernels, from its own metadata (CPU only): 64 or fewer let two blocks of 1024 threads
share a compute unit, and with them two rows of logits."""

from __future__ import annotations

import struct

import pytest

from isa.kernels.transformer_block import _hip

msgpack = pytest.importorskip("msgpack")
AMDGPU, NOTE = 0xE0, 7


def kernels():
    """{mangled name: metadata} of all code objects in the library."""
    data, at, found = _hip.LIB_PATH.read_bytes(), 0, {}
    while (at := data.find(b"\x7fELF\x02\x01\x01", at + 1)) >= 0:
        if struct.unpack_from("<H", data, at + 18)[0] != AMDGPU:
            continue
        (sections,), (size, count) = struct.unpack_from("<Q", data, at + 40), struct.unpack_from("<HH", data, at + 58)
        for i in range(count):
            header = at + sections + i * size
            if struct.unpack_from("<I", data, header + 4)[0] != NOTE:
                continue
            note = at + struct.unpack_from("<Q", data, header + 24)[0]
            name, length, _ = struct.unpack_from("<III", data, note)
            start = note + 12 + (name + 3) // 4 * 4
            for kernel in msgpack.unpackb(data[start:start + length], strict_map_key=False).get("amdhsa.kernels", []):
                found[kernel[".name"]] = kernel
    return found


@pytest.mark.parametrize("element, chunks", [("f", (2, 4, 7)), ("DF16b", (2, 4)), ("DF16_", (2, 4))], ids=["float", "bf16", "f16"])
def test_cross_entropy_shares_a_compute_unit(element, chunks):
    """Rows of up to 28672 elements in fp32, 32768 in 16-bit types, with their gradient."""
    all_kernels = kernels()
    for c in chunks:
        names = [n for n in all_kernels if f"11loss_kernelI{element}Li{c}ELi1024ELNS0_2OfE0E" in n]
        assert len(names) == 1, (element, c, names)
        kernel = all_kernels[names[0]]
        assert kernel[".vgpr_count"] + kernel.get(".agpr_count", 0) <= 64 and kernel[".vgpr_spill_count"] == 0, (c, kernel[".vgpr_count"])
