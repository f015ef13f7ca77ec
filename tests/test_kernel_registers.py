"""What the compiler made of the tree attention's kernels, from the notes in the built library: none keeps vector registers in scratch memory.
Their loops are counted by hand (waits for loads in flight), and a build of one of them that did spill gave wrong results."""
import os
import re
import struct
import subprocess

import pytest

from whisper_amd import _lib

READELF = "/opt/rocm/llvm/bin/llvm-readelf"


def code_objects(path):
    data = open(path, "rb").read()
    magic = b"__CLANG_OFFLOAD_BUNDLE__"
    for at in (m.start() for m in re.finditer(magic, data)):
        count, = struct.unpack_from("<Q", data, at + 24)
        pos = at + 32
        for _ in range(count if count < 16 else 0):
            off, size, n = struct.unpack_from("<QQQ", data, pos)
            if b"gfx950" in data[pos + 24:pos + 24 + n]:
                yield data[at + off:at + off + size]
            pos += 24 + n


@pytest.mark.skipif(not os.path.exists(READELF), reason="no llvm-readelf")
def test_tree_attention_spills_no_vector_registers(tmp_path):
    if not os.path.exists(_lib.LIB_PATH):
        import __graft_entry__
        __graft_entry__.build()
    seen = {}
    for i, obj in enumerate(code_objects(_lib.LIB_PATH)):
        f = tmp_path / f"{i}.co"
        f.write_bytes(obj)
        notes = subprocess.run([READELF, "--notes", str(f)], capture_output=True, text=True, check=True).stdout
        for kernel in re.split(r"(?m)^  - \.a", notes)[1:]:
            field = lambda name: re.search(rf"\.{name}:\s+(\S+)", kernel).group(1)  # noqa: E731
            name = re.search(r"(?m)^    \.name:\s+(\S+)", kernel).group(1)
            if re.search("tree_attention_(keys|rows)_kernel", name):
                seen[name] = int(field("vgpr_spill_count")), int(field("private_segment_fixed_size"))
    assert len(seen) >= 20 and not any(any(x) for x in seen.values()), {k: v for k, v in seen.items() if any(v)}
