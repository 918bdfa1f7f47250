"""How the paged attention's calls are cut, on the CPU (csrc/paged_plan.h): the GPU
tests' cases take the kernel and the number of splits that they are there for.
"""

import os
import subprocess

import pytest

import test_gpu_paged_joins as joins
import test_gpu_paged_uses as uses

NATIVE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "native")
STORAGES = {"F32": 0, "F16": 1, "BF16": 2, "E4M3": 3}


@pytest.fixture(scope="module")
def plan():
    subprocess.run(["make", "-s", "_build/paged_plan_of"], cwd=NATIVE, check=True)

    def cut(storage, counts, lengths, kv, group, width, page):
        given = [STORAGES[storage], kv, group, width, page, -(-max(lengths) // page), len(counts), sum(counts),
                 max(counts), max(lengths)]
        out = subprocess.run([os.path.join(NATIVE, "_build", "paged_plan_of")] + [str(n) for n in given],
                             capture_output=True, text=True, check=True, timeout=60).stdout
        return [int(n) for n in out.split()]
    return cut


def test_the_joins_cases_are_cut_as_they_say(plan):
    for given in joins.CUT_CHUNKS:
        tile_rows, splits, _, fused = plan(*given[1:], joins.PAGE)
        assert (tile_rows, splits, fused) == (128, given[0], 0), given
    for given in joins.CUT_ROWS:
        tile_rows, splits, _, fused = plan(*given[1:], joins.PAGE)
        assert tile_rows < 128 and splits == given[0] and fused == (splits <= 16), given


def test_the_captured_cases_take_every_kernel_and_join(plan):
    cuts = {}
    for name, (storage, counts, longest, kv, group, width, page, _) in uses.CAPTURED.items():
        tile_rows, splits, _, fused = plan(storage, counts, [longest] * len(counts), kv, group, width, page)
        cuts[name] = (tile_rows == 128, splits > 1, splits > 16, bool(fused))
    assert cuts == {"one-span": (False, False, False, True), "joined-in-place": (False, True, False, True),
                    "joined-after": (False, True, True, False), "fp32": (False, True, False, True),
                    "chunks": (True, False, False, False), "cut-chunks": (True, True, False, False)}


def test_the_largest_calls_are_counted_or_refused():
    subprocess.run(["make", "-s", "_build/paged_extents_check"], cwd=NATIVE, check=True)
    result = subprocess.run([os.path.join(NATIVE, "_build", "paged_extents_check")], capture_output=True, text=True,
                            timeout=60)
    assert result.returncode == 0 and "FAIL" not in result.stdout, result.stdout + result.stderr
