"""Which kernel attends over the 4-bit cache, and the room for its partial results (csrc/fourbit_choice.h), compiled
for the host: the calls that tests/test_gpu_fourbit_many.py makes for the kernel of many rows reach it."""
import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SRC = r'''
#include "fourbit_choice.h"
using namespace rtg;
extern "C" int many(int n_seq, int n_head, int hdp, int tiles, int type, long columns) {
  return for_many({n_seq, n_head, hdp, tiles}, type, columns);
}
extern "C" long parts(int n_seq, int n_head, int hdp, int tiles, long row_tiles) {
  return fmany_parts(row_tiles, {n_seq, n_head, hdp, tiles});
}
extern "C" size_t sizes(int n_seq, int n_head, int hdp, int tiles, int which) {
  const FSizes c{n_seq, n_head, hdp, tiles};
  const size_t all[] = {c.bytes(), fattn_parts_bytes(c), few_room(c) * few_part_bytes(c), many_room(c) * many_part_bytes(c),
                        (size_t)few_room(c), (size_t)many_room(c)};
  return all[which];
}
'''
F32, BF16, F16 = range(3)


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("fourbit_choice")
    (d / "c.cpp").write_text(SRC)
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "rusttorch_amd", "csrc"),
                    "-o", str(d / "libc.so"), str(d / "c.cpp")], check=True)
    got = C.CDLL(str(d / "libc.so"))
    got.many.argtypes = [C.c_int] * 5 + [C.c_long]
    got.parts.argtypes = [C.c_int] * 4 + [C.c_long]
    got.parts.restype = C.c_long
    got.sizes.restype = C.c_size_t
    return got


def tiles(capacity):
    return (capacity + 31) // 32


ANY = [c for c in range(97, 513) if c % 128 == 0 or c % 128 > 96]  # (the rule of that file's own)


# caches of tests/test_gpu_fourbit_many.py: sequences, heads, capacity, columns
@pytest.mark.parametrize("n_seq,heads,capacity,columns", [(3, 2, 200000, ANY), (5, 27, 9000, [230, 256]), (2, 1, 600000, ANY),
                                                          (1, 1, 1300000, ANY), (2, 2, 300000, ANY)])
def test_the_gpu_tests_of_many_rows_reach_their_kernel(lib, n_seq, heads, capacity, columns):
    assert n_seq * heads * capacity >= 1200000
    for n in columns:
        for hdp in (64, 128):
            for kind in (F32, BF16, F16):
                assert lib.many(n_seq, heads, hdp, tiles(capacity), kind, n), (n, hdp, kind)


def test_the_gpu_tests_of_bits_reach_both(lib):
    """240 columns of one head (test_gpu_attention_bits.py)."""
    for hdp in (64, 128):
        for kind in (F32, BF16, F16):
            assert not lib.many(1, 1, hdp, tiles(100), kind, 240) and lib.many(1, 1, hdp, tiles(1300000), kind, 240)


def test_few_columns_and_more_than_a_grid_holds(lib):
    for kind in (F32, BF16, F16):
        assert not lib.many(1, 1, 64, tiles(4000000), kind, 32)
        assert lib.many(1, 1, 64, 1, kind, 16 * 65535 + 1)


@pytest.mark.parametrize("hdp", [64, 128])
def test_room_for_partial_results(lib, hdp):
    """Within half of the cache, within 17 MB, and as many workgroups as are asked to split keys have theirs."""
    for n_seq, heads in ((1, 1), (1, 12), (3, 7), (40, 25)):
        for capacity in (1, 31, 100, 544, 1024, 1025, 4096, 10007, 100000):
            t = tiles(capacity)
            held, room, few, many, few_n, many_n = (lib.sizes(n_seq, heads, hdp, t, i) for i in range(6))
            assert held >= n_seq * heads * t * 32 * (hdp + hdp // 16 + 4) and room <= held / 2 and room <= 18 * 10 ** 6
            assert few <= room and many <= room and few_n <= 256 and many_n <= 256
            for rows in (1, 5, 100, 256):
                parts = lib.parts(n_seq, heads, hdp, t, rows)
                assert parts >= 1 and (parts == 1 or parts * rows <= many_n)
    assert lib.sizes(1, 12, hdp, tiles(100000), 4) == lib.sizes(1, 12, hdp, tiles(100000), 5) == 256
