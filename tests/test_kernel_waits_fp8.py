"""The 8-bit products' loads into LDS, which the compiler does not count, read from their assembly (built here; no GPU)."""
import os
import re
import shutil
import subprocess

import pytest
from test_kernel_waits import _blocks, _functions

from evoformer_triton_amd import build

# What holds in every step of the large kernel but its last three: a stage is asked for
ALWAYS = [("if (part == 0 && s + 3 < ns) fetch(s + 3);", "if (part == 0) fetch(s + 3);", 1), ("if (s + 3 < ns) asm volatile(", "if (true) asm volatile(", 2)]


@pytest.fixture(scope="module")
def assembly(tmp_path_factory):
    """Of the kernels as they are, and with all steps of the large one alike."""
    flags = [x for x in build.HIPCC_FLAGS if x != "-I" + build.CSRC] + next(u[2] for u in build._units() if u[0] == "fp8")
    texts = []
    for changes in ([], ALWAYS):
        csrc = tmp_path_factory.mktemp("fp8") / "csrc"
        shutil.copytree(build.CSRC, csrc)
        source = (csrc / "fp8.hip").read_text()
        for old, new, times in changes:
            assert source.count(old) == times, old
            source = source.replace(old, new)
        (csrc / "fp8.hip").write_text(source)
        out = str(csrc / "fp8.s")
        subprocess.check_call([build._hipcc(), *flags, "-I" + str(csrc), "-S", "--cuda-device-only", os.path.join(csrc, "fp8.hip"), "-o", out], stderr=subprocess.DEVNULL)
        with open(out) as f:
            texts.append(f.read())
    return texts


def _every_way(lines, step, state):
    """`step(state, instruction, by hand)` along every way through a kernel, with the least state where ways meet; called once more with it settled."""
    blocks, following = _blocks(lines)
    into, todo = {"entry": state}, ["entry"]
    while todo:
        b = todo.pop()
        out = into[b]
        for s, hand in blocks[b]:
            out = step(out, s, hand, False)
        for f in following[b]:
            new = out if f not in into else min(out, into[f])
            if f not in into or new != into[f]:
                into[f] = new
                todo.append(f)
    for b in into:
        out = into[b]
        for s, hand in blocks[b]:
            out = step(out, s, hand, True)


def test_a_stage_of_the_large_kernel_is_there_when_it_is_read(assembly):
    """Between its steps it waits for all but the eight youngest loads, the two stages after the next one: since the wait before, a whole stage of four has been asked for,
    on every way, so the next one is older than eight."""
    seen = 0
    for name, lines in _functions(assembly[1], "fp8_matmul_big"):
        def step(loads, s, hand, last):
            nonlocal seen
            wait = re.match(r"s_waitcnt\b.*vmcnt\((\d+)\)", s)
            if wait and hand:
                if last:
                    assert wait.group(1) in "08", (name, s)
                    if wait.group(1) == "8":
                        seen += 1
                        assert loads >= 4, (name, loads)
                return 0
            return min(loads + 1, 64) if s.startswith("global_load_lds_dwordx4") else loads

        _every_way(lines, step, 0)
    assert seen >= 4 * 8      # four kernels, eight steps to a turn at least


def test_a_barrier_of_the_other_kernels_finds_every_load_landed(assembly):
    """Tiles of 128 x 128 and strips: no barrier between stages is reached with a load into LDS under way."""
    seen = 0
    for kernels in ("10fp8_matmulI", "9fp8_stripI"):
        for name, lines in _functions(assembly[0], kernels):
            def step(landed, s, hand, last):
                nonlocal seen
                if re.match(r"s_waitcnt\b.*vmcnt\(0\)", s):
                    return 1
                if s.startswith("global_load_lds"):
                    return 0
                if s.startswith("s_barrier") and hand and last:
                    seen += 1
                    assert landed, name
                return landed

            _every_way(lines, step, 1)
    assert seen >= 4 + 14      # four of tiles, fourteen of strips


def test_kernels_that_load_into_lds_keep_their_registers(assembly):
    """Kernels that load into LDS keep all their registers: what is spilled would be counted with the loads."""
    spills = dict(re.findall(r"\.symbol: +(\S+)\.kd.*?\.vgpr_spill_count: +(\d+)", assembly[0], re.S))
    kernels = {n: int(c) for n, c in spills.items() if re.search(r"fp8_matmul|fp8_strip", n)}
    assert len(kernels) == 8 + 17 and not any(kernels.values()), kernels
