"""Rules of the kernel sources that no run of today's build can show broken: what
holds only by the compiler's choice of order or placement."""

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "evo2_flash_b200" / "csrc"
SOURCES = sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cuh"))


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_tensor_memory_waits_name_what_was_loaded(path):
    """A wait for tensor-memory loads orders the arithmetic on the loaded registers
    only if it names them: tmem_wait_ld does, the instruction by itself does not."""
    text = path.read_text()
    assert "tmem_wait_ld()" not in text
    if path.name != "tcgen05.cuh":
        assert "tcgen05.wait::ld" not in text
    else:
        assert re.findall(r"tcgen05\.wait::ld[^}]*", text) == [
            'tcgen05.wait::ld.sync.aligned;" ::: "memory");\n  (tmem_settle(r), ...);\n']


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_dynamic_shared_memory_is_aligned_by_itself(path):
    """Dynamic shared memory starts behind a kernel's static arrays: what is read from it
    in 16 bytes needs the alignment in its declaration, or its base rounded up."""
    text = path.read_text()
    for m in re.finditer(r"extern __shared__ (__align__\((\d+)\) )?[\w ]+ (\w+)\[\];", text):
        body = text[m.end():m.end() + 600]
        rounded = re.search(r"reinterpret_cast<uintptr_t>\(%s\) \+ (1023)\)" % m.group(3), body)
        assert rounded or int(m.group(2) or 0) >= 16, text[:m.start()].count("\n") + 1
