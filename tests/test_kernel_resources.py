"""What the built library's kernels take of a compute unit, as the compiler noted it beside them."""
import struct

import msgpack

from dooms_amd import _lib
from dooms_amd import build as B

MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def code_objects(data):
    """The gfx950 code objects of a library: bundles of (offset, size, target), one a source."""
    at = data.find(MAGIC)
    while at >= 0:
        (n,), p = struct.unpack_from("<Q", data, at + len(MAGIC)), at + len(MAGIC) + 8
        for _ in range(n):
            off, size, length = struct.unpack_from("<QQQ", data, p)
            if b"gfx950" in data[p + 24:p + 24 + length]:
                yield data[at + off:at + off + size]
            p += 24 + length
        at = data.find(MAGIC, at + 1)


def kernels(elf):
    """The kernels of a code object: the metadata note's list."""
    shoff, = struct.unpack_from("<Q", elf, 40)
    size, count = struct.unpack_from("<HH", elf, 58)
    for i in range(count):
        kind, = struct.unpack_from("<I", elf, shoff + i * size + 4)
        if kind != 7:  # notes
            continue
        p, n = struct.unpack_from("<QQ", elf, shoff + i * size + 24)
        end = p + n
        while p < end:
            name, desc, what = struct.unpack_from("<III", elf, p)
            p += 12 + (name + 3) // 4 * 4
            if what == 32:
                yield from msgpack.unpackb(elf[p:p + desc], strict_map_key=False)["amdhsa.kernels"]
            p += (desc + 3) // 4 * 4


def paged():
    _lib.lib()
    with open(B.LIB, "rb") as f:
        data = f.read()
    return {k[".name"]: k for elf in code_objects(data) for k in kernels(elf) if "paged_" in k[".name"]}


def test_the_paged_kernels_spill_no_vector_registers():
    """All but prompts over pages of codes at head dim 256, which hold a tile of 256 dims, its expansion and the queries at once."""
    found = paged()
    assert len(found) > 200
    for name, k in found.items():
        if "prefill_kernelILi256" in name and "Lb1E" in name:
            continue
        assert k[".vgpr_spill_count"] == 0 and k[".private_segment_fixed_size"] == 0, name
    decode = {n: k[".vgpr_count"] for n, k in found.items() if "paged_decode_kernelILi128" in n and n.find("Lb0ELb0E") > 0}
    assert len(decode) == 16 and max(decode.values()) <= 248, decode
