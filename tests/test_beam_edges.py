"""The beam selection's lists of candidates where they are fullest: on the CPU, a workgroup's waves restated with the library's own words,
bound and list size; on the GPU, the rows that fill them, against float64."""
import os
import subprocess

import numpy as np
import pytest

from hip_rt import Hip
from test_beam import check, reference, select

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture
def hip(gq):
    h = Hip(gq)
    yield h
    h.close()


@pytest.fixture(scope="module")
def lists(tmp_path_factory):
    """Per (logits a lane, beams, skew): the most entries of a wave, the list's size, whether the best were among them, the pattern."""
    exe = tmp_path_factory.mktemp("beam") / "beam_list_check"
    src = os.path.join(HERE, "..", "fpga-llama-gguf_amd", "csrc")
    subprocess.run([os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), "-x", "hip", "--offload-host-only", "-O2", "-std=c++17", "-ffp-contract=off", "-w",
                    "-I" + os.path.join(HERE, "..", "include"), "-I" + src, os.path.join(HERE, "beam_list_check.cpp"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe), "3"], check=True, capture_output=True, text=True).stdout
    return np.array([[int(x) for x in line.split()] for line in out.splitlines()])


def test_lists_hold_every_candidate(lists):
    """Rows that start at 16 bytes, signed zeros among them: no wave lists more than its list holds, and the best are listed in order."""
    rows = lists[lists[:, 2] == 0]
    assert len(rows) == 2 * 32
    assert (rows[:, 3] <= rows[:, 4]).all(), rows[rows[:, 3] > rows[:, 4]]
    assert rows[:, 5].all(), rows[rows[:, 5] == 0]


@pytest.mark.gpu
@pytest.mark.parametrize("beams,v", [(1, 2048), (4, 2048), (4, 40000), (8, 60000), (32, 9000)])
@pytest.mark.parametrize("what", ["one +0", "few +0", "one -0", "half"])
def test_signed_zeros_are_equal(gq, hip, beams, v, what):
    """Logits of both zeros: as equal as any others, so their order is that of the indexes."""
    print(f"[beam selection] zeros, {what}, {beams} of {v}", flush=True)
    rng = np.random.default_rng(beams + v)
    groups = 2
    x = np.full((groups, v), 0.0 if what == "one -0" else -0.0, np.float32)
    if what == "one +0":
        x[:, 7] = 0.0
    elif what == "few +0":
        x[:, 3:4 * (beams + 2):4] = 0.0
        x[:, v - 1] = 0.0
    elif what == "one -0":
        x[:, 0] = -0.0
    else:
        x[rng.random((groups, v)) < 0.5] = 0.0
    x = np.repeat(x, beams, 0)
    score = -np.arange(groups * beams, dtype=np.float32) / 4
    check(select(gq, hip, x, score, None, -1, groups, beams), reference(x, score, None, -1, groups, beams))
