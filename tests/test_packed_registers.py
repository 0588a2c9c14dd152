"""Registers of the built 16-bit backward kernels of packed attention: none of
them goes to scratch memory, in whose loops it would be read and written again
(no GPU: the library's kernels say so themselves)."""

import re
import struct

import pytest

from test_library import raw  # noqa: F401  (the fixture: the library is built)
from torch_mojo_backend.eager_kernels import LIB_PATH

msgpack = pytest.importorskip("msgpack")

NOTE = struct.pack("<I", 7)  # the owner's length, with its end; then the size, the kind 32 and the owner


def kernels():
    """{name: metadata} of the library's kernels, from the notes of its code objects."""
    data, out = open(LIB_PATH, "rb").read(), {}
    for m in re.finditer(re.escape(NOTE) + rb"(....)\x20\0\0\0AMDGPU\0\0", data, re.DOTALL):
        size, = struct.unpack("<I", m.group(1))
        notes = msgpack.unpackb(data[m.end():m.end() + size], strict_map_key=False)
        out.update({k[".name"]: k for k in notes["amdhsa.kernels"]})
    return out


@pytest.mark.parametrize("width", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("dtype", ["DF16b", "DF16_"])
def test_nothing_is_spilled(raw, dtype, width):  # noqa: F811
    found = {n: k for n, k in kernels().items() if f"10packed_bwdI{dtype}Li{width}E" in n}
    assert len(found) >= 2, "no kernels' notes in the library"
    for name, k in found.items():
        assert not k[".vgpr_spill_count"] and not k[".private_segment_fixed_size"], name
