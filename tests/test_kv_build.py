"""What the compiler made of the cache's and the beam step's kernels, read from the built library (no GPU).

Workgroups that hand data to another one of the same launch through the workspace do so with device-scope accesses (sc1): the
memory is uncached, but a CU's L1 may still hold a line that it took in before a neighbour's words of it were written, and
no wait of the writer's reaches it there."""
import functools
import os
import re
import shutil
import struct
import subprocess
import tempfile

from p0pc0rn_amd import capi

OBJDUMP = shutil.which("llvm-objdump") or "/opt/rocm/llvm/bin/llvm-objdump"
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def _objects():
    """the gfx950 code objects in the library"""
    data = open(capi.LIB_PATH, "rb").read()
    at = data.find(MAGIC)
    while at >= 0:
        n, p = struct.unpack_from("<Q", data, at + len(MAGIC))[0], at + len(MAGIC) + 8
        for _ in range(n):
            off, size, idl = struct.unpack_from("<QQQ", data, p)
            if b"gfx950" in data[p + 24:p + 24 + idl] and size:
                yield data[at + off:at + off + size]
            p += 24 + idl
        at = data.find(MAGIC, at + 1)


@functools.lru_cache(None)
def _code(kernel):
    """kernel's instantiations -> their instructions, one a line"""
    out = {}
    with tempfile.TemporaryDirectory() as d:
        f = os.path.join(d, "code.elf")
        for elf in _objects():
            if kernel.encode() not in elf:
                continue
            open(f, "wb").write(elf)
            asm = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", f], capture_output=True, text=True, check=True).stdout
            for name, body in re.findall(r"^[0-9a-f]+ <(\S+)>:\n(.*?)(?=^[0-9a-f]+ <|\Z)", asm, re.S | re.M):
                if re.match(r"_ZN2p0\d+%sI" % kernel, name):
                    out[name] = [line.split("//")[0].strip() for line in body.splitlines()]
    return out


def test_a_beam_search_is_joined_over_device_scope_accesses():
    """keys and sums are the kernels' only 8-byte accesses of global memory"""
    kernels = {**_code("beam_kernel"), **_code("beam_join_kernel")}
    assert len(kernels) == 6
    for name, code in kernels.items():
        words = [x for x in code if re.match(r"(global|flat)_(load|store)_dwordx2 ", x)]
        assert words and all(" sc1" in x for x in words), (name, [x for x in words if " sc1" not in x][:3])


def test_parts_of_an_item_are_joined_over_device_scope_accesses():
    """kv_attn_kernel's last workgroup of an item has 20 words of 8 bytes in flight; none of its loads go by `nt`, which passes by
    no cache"""
    kernels = _code("kv_attn_kernel")
    assert len(kernels) == 21
    for name, code in kernels.items():
        words = [x for x in code if re.match(r"(global|flat)_load_dwordx2 ", x) and " sc1" in x]
        stores = [x for x in code if re.match(r"(global|flat)_store_dwordx2 ", x) and " sc1" in x]
        assert len(words) >= 20 and len(stores) >= 5, (name, len(words), len(stores))
        assert not [x for x in code if re.match(r"(global|flat)_load", x) and re.search(r"\bnt\b", x)], name


def test_the_kernels_spill_no_registers():
    """not one of them does: each keeps its tile, its loads on their way and its sums in the registers that its launch bounds leave"""
    readelf = shutil.which("llvm-readelf") or "/opt/rocm/llvm/bin/llvm-readelf"
    spills = {}
    with tempfile.TemporaryDirectory() as d:
        f = os.path.join(d, "code.elf")
        for elf in _objects():
            open(f, "wb").write(elf)
            notes = subprocess.run([readelf, "--notes", f], capture_output=True, text=True, check=True).stdout
            for name, n in re.findall(r"\.name: +(_ZN2p0\d+(?:kv|beam)_\S+).*?\.vgpr_spill_count: +(\d+)", notes, re.S):
                spills[name] = int(n)
    assert len(spills) >= 21 + 24 + 6 + 8 + 12 + 6 and not any(spills.values()), {k: v for k, v in spills.items() if v}
