"""What the built kernels take of a workgroup's LDS and of scratch memory, from the descriptors in the
library's code objects."""

import re
import struct

import pytest

from conftest import ROOT

LDS = 160 * 1024  # bytes a workgroup can have
AMDGPU = 224      # an ELF file's machine


def descriptors(elf):
    """(bytes of LDS, bytes of scratch a thread) by kernel: the first two words behind each `name.kd`."""
    header, = struct.unpack_from("<Q", elf, 40)
    size, count = struct.unpack_from("<HH", elf, 58)
    sections = [struct.unpack_from("<IIQQQQII", elf, header + i * size) for i in range(count)]
    out = {}
    for _, kind, _, _, off, length, link, _ in sections:
        if kind != 11:  # exported symbols
            continue
        names = sections[link][4]
        for at in range(off, off + length, 24):
            name, _, _, section, value, _ = struct.unpack_from("<IBBHQQ", elf, at)
            text = elf[names + name:elf.index(b"\0", names + name)].decode()
            if text.endswith(".kd"):
                _, _, _, address, start, *_ = sections[section]
                out[text[:-3]] = struct.unpack_from("<II", elf, start + value - address)
    return out


@pytest.fixture(scope="module")
def kernels():
    data = (ROOT / "slm.use_amd" / "libslm_hip.so").read_bytes()
    out = {}
    for m in re.finditer(rb"\x7fELF", data):
        if m.start() and struct.unpack_from("<H", data, m.start() + 18)[0] == AMDGPU:
            out.update(descriptors(data[m.start():]))
    return out


def test_what_lies_behind_the_fixed_lds_is_aligned(kernels):
    """The part of a workgroup's LDS that a launch sizes starts behind what its kernel declares, and
    paged attention and eviction read and write 16 bytes of it at once."""
    sized = [n for n in kernels if n.startswith("slm_paged_attn") or n == "slm_paged_select"]
    assert len(sized) == 31
    assert [n for n in sized if kernels[n][0] % 16] == []


def test_the_largest_eviction_fits_in_lds(kernels):
    text = (ROOT / "slm.use_amd" / "csrc" / "runtime.cpp").read_text()
    room = int(text.split("EVICT_ROOM = ")[1].split(";")[0])
    assert room % 64 == 0
    assert kernels["slm_paged_select"][0] + room * 4 + room // 64 * 12 <= LDS


def test_the_paged_kernels_use_no_scratch_memory(kernels):
    own = [n for n in kernels if n.startswith(("slm_paged", "slm_logprobs"))]
    assert len(own) == 41 and [n for n in own if kernels[n][1]] == []
