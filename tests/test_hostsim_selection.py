"""What the CPU suite's run of the GPU tests (tests/test_hostsim_gpu_suite.py) leaves out: its list names whole node ids or
parametrisations, so that no line drops a test by the beginning of its name, and what special values and shapes are tested by
stays in the run."""
from __future__ import annotations

import os
import re
import subprocess
import sys

from tests.hostsim.build import needs_host_clang

pytestmark = needs_host_clang

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def slow():
    lines = open(os.path.join(ROOT, "tests", "hostsim", "slow_in_simulation.txt"))
    return [line.strip() for line in lines if line.strip() and not line.startswith("#")]


def collected(*args):
    run = subprocess.run([sys.executable, "-m", "pytest", "tests", "-m", "gpu", "--collect-only", "-q", "-p", "no:cacheprovider", *args],
                         cwd=ROOT, env=dict(os.environ, FLEXTRAIN_HOSTSIM="1"), capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout[-2000:] + run.stderr[-2000:]
    return [line for line in run.stdout.splitlines() if "::" in line]


def test_no_line_drops_another_test_by_its_beginning():
    ids = collected()
    functions = {i.split("[")[0] for i in ids}
    for line in slow():
        assert any(i.startswith(line) for i in ids), f"{line}: no such test"
        if "[" not in line:
            others = sorted(f for f in functions if f.startswith(line) and f != line)
            assert not others, f"{line} also drops {others}"


def test_what_stays_in_the_run():
    ids = collected(*[a for line in slow() for a in ("--deselect", line)])
    assert len(ids) >= 950
    kept = {re.split(r"::|\[", i)[1] for i in ids if "test_gpu_fp8" in i}
    for name in ("test_matmul", "test_matmul_empty", "test_matmul_nan_and_infinity_stay_in_their_rows", "test_matmul_outputs_at_any_address",
                 "test_grouped_matmul", "test_grouped_matmul_leaves_rows_behind_the_last_expert", "test_grouped_wgrad",
                 "test_quantize_grouped_columns", "test_grouped_counts_and_sources_out_of_range_stay_inside", "test_long_contractions",
                 "test_memory_that_ends_with_the_last_row", "test_experts"):
        assert name in kept, name
