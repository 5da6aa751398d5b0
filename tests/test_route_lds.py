"""Where the routing kernels' dynamic LDS begins, from the metadata of the built library:
behind the static arrays, whose size a launch rounds up to nothing.  It holds what is read
16 bytes at a time and doubles."""

import struct

import msgpack

import ien

MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def code_objects(data):
    """The gfx950 code objects of every bundle in the library."""
    at = data.find(MAGIC)
    while at >= 0:
        count, = struct.unpack_from("<Q", data, at + len(MAGIC))
        entry = at + len(MAGIC) + 8
        for _ in range(count):
            offset, size, name = struct.unpack_from("<QQQ", data, entry)
            triple = data[entry + 24:entry + 24 + name]
            entry += 24 + name
            if triple.endswith(b"gfx950") and size:
                yield data[at + offset:at + offset + size]
        at = data.find(MAGIC, entry)


def kernels(elf):
    """The metadata of a code object's kernels: its note of type 32, in msgpack."""
    first, = struct.unpack_from("<Q", elf, 0x20)
    width, count = struct.unpack_from("<HH", elf, 0x36)
    for i in range(count):
        kind, _, offset, _, _, size = struct.unpack_from("<IIQQQQ", elf, first + i * width)
        if kind != 4:  # (PT_NOTE)
            continue
        at = offset
        while at < offset + size:
            name, length, note = struct.unpack_from("<III", elf, at)
            at += 12 + -(-name // 4) * 4
            if note == 32:
                yield from msgpack.unpackb(elf[at:at + length])["amdhsa.kernels"]
            at += -(-length // 4) * 4


def test_dynamic_lds_begins_at_16_bytes():
    sizes = {k[".name"]: k[".group_segment_fixed_size"] for elf in code_objects(ien.LIB_PATH.read_bytes()) for k in kernels(elf)}
    routing = {name: size for name, size in sizes.items() if "k_route" in name or "k_plan_place" in name}
    assert len(routing) >= 4
    assert not {name: size for name, size in routing.items() if size % 16}
