"""How the attention over the paged KV cache divides its work: the host's arithmetic, compiled without a GPU."""
import ctypes
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def split(tmp_path_factory):
    """split(items, tiles, sms), run in a process of its own: an integer trap there ends that process alone."""
    d = tmp_path_factory.mktemp("paged_split")
    (d / "t.cpp").write_text('''
#include <cstdio>
#include <cstdlib>
#include "af_paged_index.h"
int main(int, char** a) { std::printf("%d", af::paged_chunk_split(std::atoll(a[1]), std::atoi(a[2]), std::atoi(a[3]))); }''')
    subprocess.run(["g++", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", "-std=c++17", "-I",
                    str(ROOT / "atomflow_b200" / "csrc"), "-o", str(d / "t"), str(d / "t.cpp")], check=True)

    def call(*args):
        r = subprocess.run([str(d / "t"), *map(str, args)], capture_output=True, text=True)
        assert r.returncode == 0, (args, r.returncode, r.stderr)
        return int(r.stdout)
    return call


@pytest.mark.parametrize("sms", [-1, 0, 1, 2, 4, 7, 8, 9, 10, 18, 36, 148])
def test_small_and_unknown_gpus_get_a_split(split, sms):
    for items in (1, 16, 1 << 30):
        for tiles in (1, 8, 16, 31, 32, 1 << 23):
            s = split(items, tiles, sms)
            assert s in (1, 2, 4, 8) and (s == 1 or (sms >= s and tiles >= 4 * s))


def test_the_split_of_148_sms(split):
    """What the rule's comment says: enough CTAs to fill the GPU once, no cluster size that does not fit."""
    assert split(16, 64, 148) == 4          # 128 new tokens of 4 sequences over 8192, 4 kv heads
    assert split(4, 64, 148) == 8 and split(1, 1000, 148) == 8
    assert split(148, 64, 148) == 1 and split(1000, 64, 148) == 1
    assert split(1, 7, 148) == 1 and split(1, 8, 148) == 2


def test_the_bound_on_the_positions_leaves_room_for_a_tile(tmp_path):
    """The caller's bound and the table's width may be as large as an int: the bound that the kernels' plans round up to
    whole tiles is not."""
    (tmp_path / "t.cpp").write_text('''
#include "af_paged_index.h"
extern "C" int bound(int max_kv, int pages, int shift) { return af::paged_kv_bound(max_kv, pages, shift); }''')
    subprocess.run(["g++", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", "-shared", "-fPIC", "-std=c++17", "-I",
                    str(ROOT / "atomflow_b200" / "csrc"), "-o", str(tmp_path / "t.so"), str(tmp_path / "t.cpp"), "-lubsan"],
                   check=True)
    bound = ctypes.CDLL(str(tmp_path / "t.so")).bound
    top, room = 2 ** 31 - 1, 2 ** 30
    for max_kv in (0, 1, 100, 4096, room - 1, room, room + 1, top - 127, top):
        for pages in (0, 1, 7, 2 ** 20, 2 ** 27, top):
            for shift in (3, 4, 8):
                want = min(max_kv or 2 ** 60, pages << shift, room)
                assert bound(max_kv, pages, shift) == want
                assert (want + 127) // 128 <= 2 ** 23
