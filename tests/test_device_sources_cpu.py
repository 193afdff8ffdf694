"""What every kernel has to keep to and no run on a healthy device shows, read from the sources."""
from __future__ import annotations

from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "halo_b200" / "csrc"


def test_the_error_word_may_be_missing():
    """A context without pinned host memory has no error word: a kernel whose wait has run out looks before it writes there."""
    writes = [(f.name, n, line.strip()) for f in sorted(CSRC.glob("*.cu*")) for n, line in enumerate(f.read_text().splitlines(), 1)
              if "atomicOr(" in line and "error_word" in line]
    assert len(writes) > 10
    assert [w for w in writes if "error_word != nullptr" not in w[2]] == []


def test_what_a_launch_names_is_not_read_in_front_of_the_kernel_before():
    """Lengths, starts and positions may have been written by the kernel before, which still runs when these kernels begin: not by loads that the compiler
    may move in front of the wait for it.  (Every other address depends on one of them.)"""
    for f in sorted(CSRC.glob("attention*")) + [CSRC / "kv_write.cu", CSRC / "rope.cu"]:
        for line in f.read_text().splitlines():
            assert not any(f"__ldg({name}" in line for name in ("r.start", "r.length", "a.positions")), (f.name, line.strip())
