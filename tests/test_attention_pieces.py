"""How the attention kernels cut an axis into pieces, compiled for the host and compared with Python's
integers, up to counts whose products pass 32 bits."""

from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "custom-3dgs-cuda_b200" / "csrc"


@pytest.fixture(scope="module")
def piece_begin(tmp_path_factory):
    d = tmp_path_factory.mktemp("pieces")
    (d / "p.cpp").write_text('#include "pieces.h"\nextern "C" int piece_begin(int n, int i, int m) '
                             "{ return gs::piece_begin(n, i, m); }\n")
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", str(CSRC), str(d / "p.cpp"), "-o",
                    str(d / "p.so")], check=True)
    return ctypes.CDLL(str(d / "p.so")).piece_begin


@pytest.mark.parametrize("count", (0, 1, 7, 128, 148, 1000, (1 << 24) - 1, 1 << 25, 29_100_000,
                                   (1 << 31) - 1024))
def test_pieces_cover_the_axis(piece_begin, count):
    for pieces in (1, 2, 3, 37, 147, 148):
        begins = [piece_begin(count, i, pieces) for i in range(pieces + 1)]
        assert begins == [count * i // pieces for i in range(pieces + 1)]


def test_the_backward_uses_them():
    """Its products of tiles and pieces pass 32 bits, where a key head has many query heads."""
    assert "KEYS ? piece_begin(tiles, piece, p.splits)" in (CSRC / "attention_backward.cu").read_text()
