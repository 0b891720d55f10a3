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
    """Per (logits a lane, beams): the most entries of a wave, the list's size, whether the best were among them, the pattern."""
    exe = tmp_path_factory.mktemp("beam") / "beam_list_check"
    src = os.path.join(HERE, "..", "fpga-llama-gguf_amd", "csrc")
    subprocess.run([os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), "-x", "hip", "--offload-host-only", "-O2", "-std=c++17", "-ffp-contract=off", "-w",
                    "-I" + os.path.join(HERE, "..", "include"), "-I" + src, os.path.join(HERE, "beam_list_check.cpp"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    return np.array([[int(x) for x in line.split()] for line in out.splitlines()])


def test_lists_hold_every_candidate(lists):
    """No wave lists more than its list holds, and the best are listed in order."""
    assert len(lists) == 2 * 32
    assert (lists[:, 2] <= lists[:, 3]).all(), lists[lists[:, 2] > lists[:, 3]]
    assert lists[:, 4].all(), lists[lists[:, 4] == 0]


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


@pytest.mark.gpu
@pytest.mark.parametrize("beams,v", [(1, 2048), (2, 2048), (4, 2048), (4, 300000), (8, 60000), (32, 9000)])
@pytest.mark.parametrize("skew", [0, 1, 2, 3])
@pytest.mark.parametrize("equal", [True, False])
def test_lanes_full_of_candidates(gq, hip, beams, v, skew, equal):
    """All logits of as many lanes of the first wave as may pass are above all others, in rows that all start `skew` floats past 16 bytes."""
    v += -(v + skew) % 4
    print(f"[beam selection] full lanes, {beams} of {v}, skew {skew}, equal {equal}", flush=True)
    rng = np.random.default_rng(beams + v)
    per = 32 if beams * -(-v // 2048) >= 192 else 8  # logits a lane
    at = np.arange(min(v, 256 * per))
    for first in range(4):
        for lanes, lane in ((n, (at + back) // 4 % 256) for n in (beams, beams + 4, beams + 5) for back in (0, skew)):  # by tokens, by lines
            x = (-5 - rng.random(v)).astype(np.float32)
            high = at[(lane >= first) & (lane < first + lanes)]
            x[high] = 2.0 if equal else (2 + rng.random(high.size)).astype(np.float32)
            x = np.repeat(x[None], beams, 0)
            score = -np.arange(beams, dtype=np.float32) / 4
            check(select(gq, hip, x, score, None, -1, 1, beams, skew), reference(x, score, None, -1, 1, beams))


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["equal", "few values", "ascending", "descending", "masked", "one left", "spikes", "zeros"])
@pytest.mark.parametrize("beams,v", [(4, 5000), (32, 9001), (1, 101), (24, 230002)])
@pytest.mark.parametrize("skew", [1, 2, 3])
def test_structured_rows_off_their_lines(gq, hip, what, beams, v, skew):
    """Rows with many equal or ordered logits, each at a place of its own in its lines: a group's beams share their logits, so they tie."""
    print(f"[beam selection] {what}, {beams} of {v}, skew {skew}", flush=True)
    rng = np.random.default_rng(3)
    x = {"equal": np.full(v, 1.25), "few values": rng.integers(-1, 2, v), "ascending": np.arange(v) / 64, "descending": -np.arange(v) / 64,
         "masked": np.where(rng.random(v) < 0.9, -np.inf, rng.standard_normal(v)), "one left": np.where(np.arange(v) == v - 1, 3.0, -np.inf),
         "spikes": np.where(np.arange(v) % 1024 == 0, 50.0, rng.standard_normal(v)),
         "zeros": np.where(rng.random(v) < 0.5, 0.0, -0.0)}[what].astype(np.float32)
    x = np.repeat(x[None], 2 * beams, 0)
    score = np.repeat(np.float32([-1.5, -2.25]), beams)
    check(select(gq, hip, x, score, None, -1, 2, beams, skew), reference(x, score, None, -1, 2, beams))


@pytest.mark.gpu
@pytest.mark.parametrize("beams,v", [(1, 100), (4, 5000), (12, 9000), (32, 40)])
@pytest.mark.parametrize("dead", ["first", "all", "nan"])
def test_ended_beams_without_a_score(gq, hip, beams, v, dead):
    """A beam whose last token is eos and whose score is -inf (or NaN): all its candidates are at -inf, ordered by their tokens."""
    rng = np.random.default_rng(beams)
    x = rng.standard_normal((2 * beams, v)).astype(np.float32)
    score = -np.arange(2 * beams, dtype=np.float32) - 1
    if dead == "first":
        score[::beams] = -np.inf
        x[1:beams] = -np.inf  # the first group has fewer candidates above -inf than winners
    else:
        score[:] = np.nan if dead == "nan" else -np.inf
    last = np.full(2 * beams, 7, np.int32)
    last[1:beams] = 3
    check(select(gq, hip, x, score, last, 7, 2, beams), reference(x, score, last, 7, 2, beams))


def _array(gq, data, **k):
    d = dict(data=data, row_stride=64, part_stride=0, n_part=1, first=0, count=16, unit_bytes=4, unit_len=1, used=0, used_stride=1)
    return gq.BeamArray(*{**d, **k}.values())


def test_arrays_past_a_launch_are_refused(gq):
    """Rows whose workgroups have 2^32 threads or more (no device is touched)."""
    lib, P, g = gq.hip_lib(), 1 << 20, 1 << 30
    for k in (dict(count=64, unit_bytes=g, row_stride=64 * g), dict(n_part=2, count=32, unit_bytes=g, row_stride=64 * g, part_stride=32 * g),
              dict(n_part=65535, count=257, unit_bytes=4096, row_stride=257 << 12, part_stride=257 << 13)):
        assert lib.gemvq_beam_reorder_static((gq.BeamArray * 1)(_array(gq, P, **k)), 1, P, 1, 2 if k.get("n_part") != 2 else 1, 0) == gq.EINVAL, k


@pytest.mark.gpu
def test_arrays_that_fill_several_launches(gq, hip):
    """Two arrays of two rows of 33 GiB, whose workgroups do not fit one launch (of each the first 12288 bytes are in use), and small
    ones before, between and behind them."""
    rng = np.random.default_rng(2)
    row, page = 33 << 30, 4096
    try:
        big = [hip.alloc(2 * row) for _ in range(2)]
    except AssertionError:
        pytest.skip("132 GiB of device memory are not free")
    small = [rng.integers(0, 1 << 30, (2, 16)).astype(np.int32) for _ in range(3)]
    large = [rng.integers(0, 256, (2, 4 * page)).astype(np.uint8) for _ in big]
    for b, x in zip(big, large):
        for i in range(2):
            hip.write(b + i * row, x[i])
    used = hip.upload(np.int32([3, 3]))
    at = [hip.upload(x) for x in small]
    arrays = [_array(gq, at[0])]
    for b, p in zip(big, at[1:]):
        arrays += [_array(gq, b, row_stride=row, count=row // page, unit_bytes=page, used=used), _array(gq, p)]
    gq.beam_reorder_static(arrays, hip.upload(np.int32([1, 1])), 1, 2)
    for x, p in zip(small, at):
        assert np.array_equal(hip.download(p, x.shape, np.int32), x[[1, 1]])
    for b, x in zip(big, large):
        assert np.array_equal(hip.download(b, (4 * page,), np.uint8), np.concatenate([x[1, :3 * page], x[0, 3 * page:]]))
        assert np.array_equal(hip.download(b + row, (4 * page,), np.uint8), x[1])
