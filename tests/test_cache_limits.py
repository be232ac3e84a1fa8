"""Host side of the cache's long-context operators at the edges of their range,
without a GPU (no call here launches a kernel): counts that pass 32 bits,
empty calls, launches beyond what the device takes, arrays that overlap."""
from __future__ import annotations

import ctypes as C
import pathlib
import subprocess

import pytest

from flashmlx_amd import _lib

ROOT = pathlib.Path(__file__).resolve().parents[1]


def test_pieces_cover_the_keys():
    """The pieces that own keys are dealt to, for batches up to the limit of
    2^36 own positions (tests/c_abi/piece_check.cpp, built by
    __graft_entry__.build())."""
    prog = ROOT / "tests" / "c_abi" / "_build" / "piece_check"
    assert prog.exists(), f"{prog} missing: run __graft_entry__.build()"
    p = subprocess.run([str(prog)], capture_output=True, text=True, timeout=60)
    assert p.returncode == 0, p.stdout + p.stderr


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _shape(dtype=_lib.FMX_BF16, B=2, L=1, nh=8, nkv=2, hd=128, scale=0.1):
    return C.byref(_lib.FmxAttentionShape(dtype, B, L, nh, nkv, hd, scale))


@pytest.mark.parametrize("kw", [dict(B=0), dict(L=0), dict(B=0, L=0), dict(B=0, L=1 << 24, nh=65535, nkv=1),
                                dict(B=0, L=40), dict(L=0, B=1 << 24)], ids=str)
def test_empty_calls_need_no_workspace(lib, kw):
    """No sequences or no queries: 0 bytes (the process ended before)."""
    for P, S in ((0, 0), (5, 0), (0, 8), (5, 8), (20000, 9000)):
        if S:
            assert lib.fmx_attention_scored_workspace_size(_shape(**kw), S) == 0
        assert lib.fmx_attention_shared_prefix_workspace_size(_shape(**kw), P, S) == 0
