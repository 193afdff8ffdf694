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
