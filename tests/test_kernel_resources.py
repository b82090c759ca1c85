"""CPU: what the compiler gave the kernels of the built library (the code objects' own metadata: registers, spills, scratch)."""
import struct

import pytest

from rise_sdf_amd import _lib

msgpack = pytest.importorskip("msgpack")


def code_objects(blob):
    """ELF images of the clang offload bundles in a shared object: magic, number of entries, (offset, size, length of the target's name, name)."""
    magic, at = b"__CLANG_OFFLOAD_BUNDLE__", 0
    while (at := blob.find(magic, at)) >= 0:
        count, p = struct.unpack_from("<Q", blob, at + len(magic))[0], at + len(magic) + 8
        for _ in range(count):
            offset, size, length = struct.unpack_from("<QQQ", blob, p)
            name = blob[p + 24:p + 24 + length]
            p += 24 + length
            if b"gfx950" in name and size:
                yield blob[at + offset:at + offset + size]
        at += len(magic)


def kernels(elf):
    """Kernel records of a code object's metadata note (type 32, msgpack)."""
    shoff, = struct.unpack_from("<Q", elf, 0x28)
    shentsize, shnum = struct.unpack_from("<HH", elf, 0x3A)
    for i in range(shnum):
        kind, = struct.unpack_from("<I", elf, shoff + i * shentsize + 4)
        offset, size = struct.unpack_from("<QQ", elf, shoff + i * shentsize + 24)
        p = offset
        while kind == 7 and p < offset + size:                                  # SHT_NOTE
            namesz, descsz, note = struct.unpack_from("<III", elf, p)
            desc = p + 12 + (namesz + 3) // 4 * 4
            if note == 32:
                yield from msgpack.unpackb(elf[desc:desc + descsz])["amdhsa.kernels"]
            p = desc + (descsz + 3) // 4 * 4


@pytest.fixture(scope="module")
def records():
    with open(_lib.SO_PATH, "rb") as f:
        blob = f.read()
    return [k for elf in code_objects(blob) for k in kernels(elf)]


def test_every_unit_is_there(records):
    for name in ("lookup_kernel", "head_walk_kernel", "linear_fwd_kernel", "layer_bwd_kernel", "specular_kernel"):
        assert any(name in k[".name"] for k in records), name


def test_layer_weight_gradient_does_not_spill(records):
    """Its row loop has no room for scratch traffic: 9 spilled registers cost 1.8 times its time."""
    mine = [k for k in records if "linear_bwd_weight_kernel" in k[".name"]]
    assert len(mine) == 8                     # widths of 32, 64, 96 and 128 in both precisions
    for k in mine:
        assert k[".vgpr_spill_count"] == 0 and k[".private_segment_fixed_size"] == 0, (k[".name"], k[".vgpr_spill_count"])
