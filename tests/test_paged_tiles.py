"""The division of a paged batch into tiles (tritify_amd/csrc/kt_paged.h), built for the host: which sequence a tile is given,
for row starts within the rules and for any others. A tile before its sequence's first would reach rows before it."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def tile_seq(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("paged") / "paged_host.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", "-I", os.path.join(ROOT, "tritify_amd", "csrc"),
                    "-I", os.path.join(ROOT, "include"), "-I", "/opt/rocm/include", os.path.join(ROOT, "tests", "paged_host.cpp"), "-o", so],
                   check=True)
    f = C.CDLL(so).paged_tile_seq
    f.restype, f.argtypes = C.c_int, [C.c_void_p] + [C.c_int] * 6 + [C.POINTER(C.c_int)]

    def call(row_start, tokens, t, mul, step, per):
        rs, first = np.ascontiguousarray(row_start, dtype=np.int32), C.c_int(-99)
        b = f(rs.ctypes.data, len(rs) - 1, tokens, t, mul, step, per, C.byref(first))
        return b, first.value

    return call


# the units of the append (rows in blocks of 16, two more a sequence) and of the attention (16 columns, rep a row)
FORMS = [(1, 16, 2), (1, 16, 0), (7, 16, 0), (20, 16, 0)]


@pytest.mark.parametrize("mul,step,per", FORMS)
@pytest.mark.parametrize("seqs", [1, 3, 64, 65, 300])
def test_every_tile_of_a_sequence_is_found(tile_seq, seqs, mul, step, per):
    g = np.random.default_rng(seqs)
    rows = np.where(g.random(seqs) < 0.4, 0, g.integers(0, 40, seqs))
    rs = np.concatenate([[0], np.cumsum(rows)])
    begin = rs[:-1] * mul // step + per * np.arange(seqs)
    for t in range(int(rs[-1]) * mul // step + per * seqs):
        b, first = tile_seq(rs, int(rs[-1]), t, mul, step, per)
        want = int(np.flatnonzero(begin <= t)[-1])
        assert (b, first) == (want, begin[want]), t


@pytest.mark.parametrize("mul,step,per", FORMS)
def test_no_tile_is_before_its_sequences_first(tile_seq, mul, step, per):
    """Row starts that decrease, start below 0 or end past the rows: a sequence that begins at or before the tile, or none."""
    g = np.random.default_rng(3)
    cases = [([0, 90, 40, 60], 90), ([90, 0, 90, 30, 90], 90), ([0, 90, 89, 88, 87, 90], 90), ([-5, 200, -7, 50], 90), ([9, 3], 90)]
    cases += [(g.integers(-20, 400, size=n + 1), 380) for n in (2, 5, 63, 64, 65, 130, 200)]
    for rs, tokens in cases:
        rs = np.asarray(rs)
        begin = np.clip(rs[:-1], 0, tokens) * mul // step + per * np.arange(len(rs) - 1)
        for t in range(tokens * mul // step + per * (len(rs) - 1)):
            b, first = tile_seq(rs, tokens, t, mul, step, per)
            assert b == -1 or (first == begin[b] and first <= t), (rs.tolist(), t, b, first)
