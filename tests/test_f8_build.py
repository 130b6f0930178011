"""What the compiler made of the 8-bit operators' kernels, read from the built library (no GPU): the products keep a tile's sums, their
fragments and the products on their way to the sums in registers, and none spills one."""
import os
import re
import shutil
import subprocess
import tempfile

from tests.test_kv_build import _code, _objects

READELF = shutil.which("llvm-readelf") or "/opt/rocm/llvm/bin/llvm-readelf"


def test_the_kernels_spill_no_registers():
    spills = {}
    with tempfile.TemporaryDirectory() as d:
        f = os.path.join(d, "code.elf")
        for elf in _objects():
            open(f, "wb").write(elf)
            notes = subprocess.run([READELF, "--notes", f], capture_output=True, text=True, check=True).stdout
            for name, n in re.findall(r"\.name: +(_ZN2p0\d+(?:f8_|rope_)\S+).*?\.vgpr_spill_count: +(\d+)", notes, re.S):
                spills[name] = int(n)
    assert len(spills) == 3 + 6 + 54 + 27 + 14 + 12 and not any(spills.values()), {k: v for k, v in spills.items() if v}


def test_slices_are_joined_over_device_scope_accesses():
    """the sums of a tile's slices are the tile kernel's only 8-byte accesses of global memory but for the 16-bit results' stores"""
    kernels = _code("f8_tile_kernel")
    assert len(kernels) == 14
    for name, code in kernels.items():
        if "F8TileILi2ELi4ELi8ELi4ELi2E" in name:   # the widest tile takes no slices
            assert not any(" sc1" in x for x in code), name
            continue
        loads = [x for x in code if re.match(r"(global|flat)_load_dwordx2 ", x)]
        stores = [x for x in code if re.match(r"(global|flat)_store_dwordx2 ", x) and " sc1" in x]
        assert len(loads) >= 8 and all(" sc1" in x for x in loads) and len(stores) >= 8, (name, len(loads), len(stores))
