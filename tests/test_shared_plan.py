"""How decode behind a shared prefix is cut (shared_plan in csrc/tile_table.h), compiled for the
CPU: what every plan has to hold, and the plans of the calls that reach the kernels' rarer paths
(PLANS, run on the GPU by test_gpu_decode_shared_plans.py)."""
import ctypes
import os
import random
import subprocess
from collections import namedtuple

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "inkling-fa4-relative-attention_amd", "csrc")
SRC = r"""
#include "tile_table.h"
extern "C" void plan(const int64_t* a, int64_t* out) {
  const ifa4::SharedPlan s = ifa4::shared_plan(a[0], a[1], a[2], a[3], a[4], a[5], a[6], a[7]);
  const int64_t x[7] = {s.prefix_keys, s.chunk_keys, s.prefix_chunks, s.row_tiles,
                        s.prefix_blocks, s.own_chunks, s.own_first};
  for (int i = 0; i < 7; ++i) out[i] = x[i];
}
"""
Plan = namedtuple("Plan", "prefix_keys chunk_keys prefix_chunks row_tiles prefix_blocks own_chunks "
                          "own_first")


def _starts(chunk, window, parts):
    """Lengths whose window starts in the given parts: at their edges, next to them, and at the
    edges of their second tile."""
    return [chunk * m + off + window + 1 for m in parts for off in (0, 1, 63, 64, 65, chunk - 1)]


# name: lengths, prefix, query and kv heads, window, bias extent
PLANS = {
    # pieces of two tiles under a window, which begins and ends inside them; 259 parts
    "windowed_pieces_of_two_tiles": (
        _starts(128, 1023, (3, 100, 240, 246)) + [33068, 32769, 32768, 500, 1, 0], 32768, 8, 2, 1023, 128),
    # 515 parts: rows whose first part is left of, across and right of the 256th
    "windowed_parts_past_256": (
        _starts(64, 511, (100, 250)) + [16384 + n for n in (255, 500, 511, 512, 513, 600)] + [33068, 32769],
        32768, 4, 1, 511, 128),
    # 343 parts of one row
    "parts_past_256": ([131072 + 50], 131072, 2, 1, -1, 128),
}


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(SRC)
    out = str(d / "plan.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", f"-I{CSRC}",
                    str(d / "plan.cpp"), "-o", out], check=True)
    lib = ctypes.CDLL(out)

    def call(batch, kv_heads, group, prefix, max_k, window, extent, slots=512):
        args = (ctypes.c_int64 * 8)(batch, kv_heads, group, prefix, max_k, window, extent, slots)
        got = (ctypes.c_int64 * 7)()
        lib.plan(args, got)
        return Plan(*got)
    return call


def test_what_every_plan_holds(plan):
    rng = random.Random(5)
    for _ in range(4000):
        batch, kv_heads = int(2 ** rng.uniform(0, 10)), rng.choice([1, 2, 3, 4, 5, 8, 16])
        group = rng.choice([1, 2, 3, 4, 8, 16])
        prefix = int(2 ** rng.uniform(0, 20)) if rng.random() < 0.95 else 0
        max_k = prefix + int(2 ** rng.uniform(0, 14)) if rng.random() < 0.9 else rng.randint(0, prefix)
        window = rng.choice([-1, -1, 0, 63, 64, 511, 1023, 4096, 100000])
        args = batch, kv_heads, group, prefix, max_k, window, rng.choice([0, 1, 128, 1024, 4096])
        s = plan(*args)
        # the prefix: whole tiles, in chunks of whole tiles, the last one not empty
        assert s.prefix_keys == min(prefix, max_k) // 64 * 64, (args, s)
        assert s.chunk_keys >= 64 and s.chunk_keys % 64 == 0, (args, s)
        assert s.prefix_chunks == -(-s.prefix_keys // s.chunk_keys), (args, s)
        # a workgroup for each of its pieces, and as many for every XCD
        assert s.row_tiles == -(-batch * group // 128), (args, s)
        assert s.prefix_blocks == -(-s.prefix_chunks * kv_heads // 8) * 8 * s.row_tiles, (args, s)
        # keys past it: pieces of at least one round of 128 keys
        rounds = -(-(max_k - s.prefix_keys) // 128)
        assert (s.own_chunks > 0) == (rounds > 0) and s.own_chunks <= rounds, (args, s)
        assert s.own_first >= 0 and (s.own_chunks > 0 or s.own_first == 0), (args, s)


@pytest.mark.parametrize("name,chunk,parts", [("windowed_pieces_of_two_tiles", 128, 259),
                                              ("windowed_parts_past_256", 64, 515),
                                              ("parts_past_256", 384, 343)])
def test_plans_of_the_rarer_paths(plan, name, chunk, parts):
    lens, prefix, hq, hkv, window, extent = PLANS[name]
    s = plan(len(lens), hkv, hq // hkv, prefix, max(lens), window, extent)
    assert s.chunk_keys == chunk and s.prefix_chunks + s.own_chunks == parts, s
    if window >= 0:  # the row's first part: some left of the 256th, some past it
        first = [max(0, n - 1 - window) // chunk for n in lens]
        assert min(first) < 255 and (parts < 512 or max(first) >= 256)
