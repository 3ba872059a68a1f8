"""No kernel of the per-token objectives or the optimizer step keeps registers in memory (a spill, or accumulators that the
compiler left in an array, cost whole factors that no numerics test would notice): from the built library's own metadata."""
import os
import re
import shutil
import struct
import subprocess

import pytest

from maester_amd import _lib

READELF = shutil.which("llvm-readelf") or "/opt/rocm/llvm/bin/llvm-readelf"
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def _kernels(path, tmp_path):
    """{kernel: (vector registers spilled, bytes of memory per lane)} of every code object in the library."""
    data = open(path, "rb").read()
    out = {}
    for m in re.finditer(MAGIC, data):
        at = m.start() + len(MAGIC)
        entries, = struct.unpack_from("<Q", data, at)
        at += 8
        for _ in range(entries):
            offset, size, length = struct.unpack_from("<QQQ", data, at)
            target = data[at + 24: at + 24 + length]
            at += 24 + length
            if b"gfx950" not in target:
                continue
            elf = tmp_path / "code.elf"
            elf.write_bytes(data[m.start() + offset: m.start() + offset + size])
            notes = subprocess.run([READELF, "--notes", str(elf)], capture_output=True, text=True, check=True).stdout
            for k in notes.split("- .agpr_count:")[1:]:
                field = {n: re.search(r"\.%s:\s+(\S+)" % n, k).group(1) for n in ("name", "vgpr_spill_count", "private_segment_fixed_size")}
                out[field["name"]] = int(field["vgpr_spill_count"]), int(field["private_segment_fixed_size"])
    return out


@pytest.mark.skipif(not os.path.exists(READELF), reason="llvm-readelf not installed")
def test_nothing_lives_in_memory(tmp_path):
    _lib.lib()
    kernels = _kernels(_lib.LIB_PATH, tmp_path)
    for name, count in (("linear_logprobs_kernel", 32), ("linear_grads_kernel", 21), ("token_logprobs_fwd_kernel", 8),
                        ("token_logprobs_bwd_kernel", 4), ("adamw_kernel", 2), ("grad_norm_kernel", 1)):
        mine = {k: v for k, v in kernels.items() if name in k}
        assert len(mine) == count, (name, len(mine))
        assert all(v == (0, 0) for v in mine.values()), {k: v for k, v in mine.items() if v != (0, 0)}
