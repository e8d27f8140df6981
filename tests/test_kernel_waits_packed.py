"""Packed attention's loads into LDS, which the compiler does not count, read from its kernels' assembly (built here; no GPU)."""
import os
import re
import subprocess

import pytest
from test_kernel_waits import _functions
from test_kernel_waits_fp8 import _every_way

from evoformer_triton_amd import build

INTO_LDS = re.compile(r"buffer_load_dword\w* .*\blds\b")


@pytest.fixture(scope="module", params=[32, 64, 96, 128])
def assembly(request, tmp_path_factory):
    texts = {}
    for name in ("packed_mfma", "packed_dkdv"):
        unit = next(u for u in build._units() if u[0] == f"{name}_d{request.param}")
        out = str(tmp_path_factory.mktemp("packed") / f"{name}.s")
        subprocess.check_call([build._hipcc(), *build.HIPCC_FLAGS, *unit[2], "-S", "--cuda-device-only", os.path.join(build.CSRC, unit[1]), "-o", out], stderr=subprocess.DEVNULL)
        with open(out) as f:
            texts[name] = f.read()
    return request.param, texts


def test_the_loops_wait_by_hand_alone(assembly):
    """A wait of the compiler's in the loop, for an operand that was asked for before it or that is kept in memory, would be one for the next stage's loads too."""
    seen = 0
    for text in assembly[1].values():
        for name, lines in _functions(text, "packed_(?:fwd|dq|dkdv)"):
            loops, where, hand = {}, None, False
            for line in lines:
                if re.match(r"\.LBB\w+:|; %bb", line):
                    header = re.search(r"in Loop: Header=(BB\w+) Depth=1", line) or re.search(r"Parent Loop (BB\w+) Depth=1", line)
                    where = header.group(1) if header else re.match(r"\.L(BB\w+):", line).group(1) if "Loop Header: Depth=1" in line else None
                elif re.search(r"Parent Loop (BB\w+) Depth=1", line) and where is not None:      # (of a loop within it, on the line after its label)
                    where = re.search(r"Parent Loop (BB\w+) Depth=1", line).group(1)
                hand = "#ASMSTART" in line or (hand and "#ASMEND" not in line)
                if where and not line.lstrip().startswith(";"):
                    loops.setdefault(where, []).append((line.strip(), hand))
            stages = [body for body in loops.values() if any(INTO_LDS.search(s) for s, _ in body)]
            assert len(stages) == 1, (name, len(stages))
            assert any("s_barrier" in s for s, _ in stages[0]), name
            assert not [s for s, by_hand in stages[0] if "vmcnt" in s and not by_hand], name
            assert not [s for s, _ in stages[0] if s.startswith("scratch_")], name
            seen += 1
    assert seen == 2 * 9        # two types; forward, dQ, dK and dV, of one group, of two, in parts


def test_a_stage_is_there_when_it_is_read(assembly):
    """No barrier is reached with a load into LDS asked for since the last wait; a wait leaves none on its way but those of the stages that are asked for further ahead, each of which has been asked for as a
    whole since the wait before."""
    ahead = {32: {1: 2, 2: 1}, 64: {1: 0, 2: 0}, 96: {1: 0, 2: 0}, 128: {1: 0, 2: 0}}[assembly[0]]      # such stages, by groups of waves
    barriers = waits = 0
    for kernel, text in assembly[1].items():
        for name, lines in _functions(text, "packed_(?:fwd|dq|dkdv)"):
            left = 0 if kernel == "packed_dkdv" else ahead[int(re.search(r"IDF16[b_]Li(\d)", name).group(1))]

            def landed(state, s, hand, last):
                nonlocal barriers
                if hand and re.match(r"s_waitcnt\b.*vmcnt", s):
                    return 1
                if hand and s.startswith("s_barrier") and last:
                    barriers += 1
                    assert state, name
                return 0 if INTO_LDS.match(s) else state

            def whole(loads, s, hand, last):
                nonlocal waits
                wait = re.match(r"s_waitcnt\b.*vmcnt\((\d+)\)", s)
                if wait and hand:
                    n = int(wait.group(1))
                    if last and n:
                        waits += 1
                        assert left and n % left == 0 and loads >= n // left, (name, s, loads)
                    return 0
                return min(loads + 1, 64) if INTO_LDS.match(s) else loads

            _every_way(lines, landed, 1)
            _every_way(lines, whole, 0)
    assert barriers >= 2 * 9 and (waits >= 2 * 6) == (assembly[0] == 32)
