"""The skinny form's scratch (csrc/skinny_plan.cuh, host arithmetic alone): a call's covers every block of 64 rows that it is
cut into, the last one of fewer rows included."""
import ctypes
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "scala-torch_b200", "csrc")
SOURCE = """
#include "skinny_plan.cuh"
using namespace stb;
extern "C" unsigned long long block_bytes(int M, int N, int K, int sms) {
  const SkinnyPlan q = skinny_plan_of(M, N, K, sms);
  return q.x3_bytes + q.part_bytes;
}
extern "C" int pieces(int M, int N, int K, int sms) { return skinny_plan_of(M, N, K, sms).pmax; }
extern "C" unsigned long long call_bytes(int M, int N, int K, int sms) { return skinny_bytes_of(M, N, K, sms); }
extern "C" unsigned long long bytes_up_to(int rows, int N, int K, int sms) { return skinny_bytes_up_to(rows, N, K, sms); }
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    where = tmp_path_factory.mktemp("plan")
    (where / "plan.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, str(where / "plan.cpp"), "-o", str(where / "plan.so")], check=True)
    lib = ctypes.CDLL(str(where / "plan.so"))
    for name in ("block_bytes", "call_bytes", "bytes_up_to"):
        getattr(lib, name).restype = ctypes.c_ulonglong
    return lib


SHAPES = [(6144, 768), (2048, 2048), (1024, 4096), (4096, 1024), (2560, 2560), (4864, 896), (128, 64), (131072, 128), (200, 136), (8192, 28672)]


def test_a_last_block_of_few_rows_may_take_more_than_a_whole_one(plan):
    assert plan.pieces(64, 6144, 768, 148) == 5 and plan.pieces(32, 6144, 768, 148) == 13
    for N, K, rows in ((6144, 768, 32), (2048, 2048, 25), (1024, 4096, 26), (4096, 1024, 28), (2560, 2560, 30), (4864, 896, 27)):
        assert plan.block_bytes(rows, N, K, 148) > plan.block_bytes(64, N, K, 148)


@pytest.mark.parametrize("sms", [148, 1, 20, 132])
def test_a_calls_scratch_covers_each_of_its_blocks(plan, sms):
    rng = random.Random(sms)
    shapes = SHAPES + [(rng.randrange(128, 20000), 8 * rng.randrange(8, 2000)) for _ in range(10)]
    for N, K in shapes:
        for M in [*range(1, 200), 255, 256, 1000, 1056, 8191]:
            blocks = [min(64, M - m) for m in range(0, M, 64)]
            assert plan.call_bytes(M, N, K, sms) == max(plan.block_bytes(m, N, K, sms) for m in set(blocks))


def test_scratch_up_to_a_row_count_serves_every_call_of_fewer(plan):
    for N, K in SHAPES:
        for rows in (1, 2, 15, 16, 17, 31, 32, 33, 40, 63, 64, 65, 96, 500):
            most = rows if rows < 64 else 4 * 64 + 63  # from 64 rows on a call of any length
            need = max(plan.call_bytes(m, N, K, 148) for m in range(1, most + 1))
            assert plan.bytes_up_to(rows, N, K, 148) == need
