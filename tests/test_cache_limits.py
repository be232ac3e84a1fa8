"""Host side of the cache's long-context operators at the edges of their range,
without a GPU (no call here launches a kernel): counts that pass 32 bits,
empty calls, launches beyond what the device takes, arrays that overlap."""
from __future__ import annotations

import pathlib
import subprocess

ROOT = pathlib.Path(__file__).resolve().parents[1]


def test_pieces_cover_the_keys():
    """The pieces that own keys are dealt to, for batches up to the limit of
    2^36 own positions (tests/c_abi/piece_check.cpp, built by
    __graft_entry__.build())."""
    prog = ROOT / "tests" / "c_abi" / "_build" / "piece_check"
    assert prog.exists(), f"{prog} missing: run __graft_entry__.build()"
    p = subprocess.run([str(prog)], capture_output=True, text=True, timeout=60)
    assert p.returncode == 0, p.stdout + p.stderr
