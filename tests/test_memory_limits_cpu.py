"""The memory operators' queries at sizes beyond what the calls take: they answer 0, and the process lives. Each
runs in a process of its own, which a division by zero would end."""
import subprocess
import sys

import pytest

from conftest import ROOT

QUERY = """
import ctypes as C, sys
sys.path.insert(0, {package!r})
from t8b import _lib
lib = _lib.lib()
for sequences, steps, channels in {sizes!r}:
    q = _lib.Sequences(sequences=sequences, steps=steps, channels=channels)
    got = [lib.t8b_causal_conv_workspace(C.byref(q), 4), lib.t8b_selective_scan_saved(C.byref(q), 1, 16)]
    got += [lib.t8b_selective_scan_workspace(C.byref(q), 1, 16, backward) for backward in (0, 1)]
    print(*got)
"""


def answers(sizes):
    source = QUERY.format(package=str(ROOT / "tekken8-agent_b200"), sizes=sizes)
    done = subprocess.run([sys.executable, "-c", source], capture_output=True, text=True)
    assert done.returncode == 0, (done.returncode, done.stderr[-500:])
    return [[int(v) for v in line.split()] for line in done.stdout.splitlines()]


@pytest.mark.parametrize("sizes", [
    (1, 8, 1 << 32), (1, 8, 1 << 34), (1, 8, (1 << 20) + 1), (1, 1 << 32, 8), (1, 1 << 31, 8), (1, (1 << 30) + 1, 8), ((1 << 30) + 1, 8, 8),
    (1 << 32, 8, 8), (1, 8, (1 << 63) - 1), (1, (1 << 63) - 1, 8), ((1 << 63) - 1, 8, 8), (1, -1, 8), (-1, 8, 8), (1, 8, -8),
])
def test_sizes_that_no_call_takes(sizes):
    assert answers([sizes]) == [[0, 0, 0, 0]]


def test_the_largest_sizes():
    """The limits themselves are counted: states of every eighth step, one row of (width + 1) sums at least."""
    largest = [(1, 1 << 30, 1), (1 << 30, 1, 1), (1, 1, 1 << 20), (3, 7, 1 << 20), (1 << 15, 1 << 15, 8)]
    for (sequences, steps, channels), (conv, saved, _, backward) in zip(largest, answers(largest)):
        assert conv >= 4 * 5 * channels
        assert saved == sequences * -(-steps // 8) * 16 * channels
        assert backward >= 4 * (sequences * steps * 2 * 16 + channels * 18)
