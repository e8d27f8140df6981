"""The loads into LDS of packed attention's kernel for few queries, read from its assembly (built here; no GPU).

Each wave fills a buffer of keys and one of values of its own, in turn, and waits for them by counts: there is no barrier that would cover a wait too few.
"""
import re
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest
from test_kernel_waits import _blocks, _functions

from evoformer_triton_amd import build

INTO_LDS = re.compile(r"buffer_load_dword\w* .*\blds\b")


MORE = "const bool more = next < key_to;   // (uniform)"      # (of which five branches of a step are: followed one by one they would be ways that no wave takes)
END, NEXT = "if (!more) break;", "key = next;"


# The kernels as they are, with every step one that goes on (and then waits for everything and ends, or not), and with one whose first step is its last
CHANGES = ([], [(MORE, "const bool more = true;"), (END, ""), (NEXT, NEXT + " if (key >= key_to) { wait_loads(); break; }")], [(MORE, "const bool more = false;")])


@pytest.fixture(scope="module")
def assembly(tmp_path_factory):
    def compiled(job):
        D, changes, csrc = job
        unit = next(u for u in build._units() if u[0] == f"packed_few_d{D}")
        shutil.copytree(build.CSRC, csrc)
        source = (csrc / unit[1]).read_text()
        for old, new in changes:
            assert source.count(old) == 1, old
            source = source.replace(old, new)
        (csrc / unit[1]).write_text(source)
        flags = [x for x in build.HIPCC_FLAGS if x != "-I" + build.CSRC]
        subprocess.check_call([build._hipcc(), *flags, "-I" + str(csrc), *unit[2], "-S", "--cuda-device-only", str(csrc / unit[1]), "-o", str(csrc / "kernel.s")], stderr=subprocess.DEVNULL)
        found = list(_functions((csrc / "kernel.s").read_text(), "packed_few"))
        assert len(found) == 2 * 2 * 2 * 2         # types; in parts or not; few waves or many; 16 columns or 32
        return found

    root = tmp_path_factory.mktemp("packed_few")
    jobs = [(D, changes, root / f"{D}-{i}") for D in (32, 64, 96, 128) for i, changes in enumerate(CHANGES)]
    with ThreadPoolExecutor(4) as pool:
        done = list(pool.map(compiled, jobs))
    return {D: done[3 * i:3 * i + 3] for i, D in enumerate((32, 64, 96, 128))}


@pytest.fixture(params=[32, 64, 96, 128])
def kernels(request, assembly):
    return request.param, assembly[request.param]


def _check_all(name, lines, pieces):
    """Every state that a wave can be in, along every way.  A state: the loads into LDS that may be under way, oldest first (K and V: pieces of keys and of values, which are asked for in turn); how many have been
    asked for, modulo both buffers'; whether reads of the keys, and of the values, may not have returned.  -> (reads of keys, reads of values, loads) met"""
    blocks, following = _blocks(lines)
    into, todo, met = {"entry": {("", 0, False, False)}}, ["entry"], [0, 0, 0]

    def step(state, s):
        under_way, asked, keys, values = state
        if INTO_LDS.match(s):
            kind = "K" if asked < pieces else "V"
            assert not (keys if kind == "K" else values), (name, s, "asked for before the reads of what lies there have returned")
            met[2] += 1
            return under_way + kind, (asked + 1) % (2 * pieces), keys, values
        if s.startswith("s_waitcnt"):
            vm = re.search(r"vmcnt\((\d+)\)", s)
            if vm and int(vm.group(1)) < len(under_way):
                under_way = under_way[len(under_way) - int(vm.group(1)):]
            if "lgkmcnt(0)" in s:
                keys = values = False
        elif s.startswith("ds_read_b64_tr"):
            assert "V" not in under_way, (name, s, under_way)
            met[1] += 1
            values = True
        elif s.startswith("ds_read_b128"):
            assert "K" not in under_way, (name, s, under_way)
            met[0] += 1
            keys = True
        elif s.startswith("s_barrier"):
            assert not under_way, (name, under_way)
        return under_way, asked, keys, values

    while todo:
        b = todo.pop()
        states = into[b]
        for s, _ in blocks[b]:
            states = {step(x, s) for x in states}
        for f in following[b]:
            if not states <= into.get(f, set()):
                into[f] = into.get(f, set()) | states
                todo.append(f)
    return met


def _pieces(D):
    return {32: 2, 64: 4}.get(D, 8)


def test_keys_and_values_are_there_when_they_are_read(kernels):
    D, (_, on, last) = kernels
    for found in (on, last):
        for name, lines in found:
            met = _check_all(name, lines, _pieces(D))
            assert all(met), (name, met)


def test_a_wait_too_few_would_be_seen(kernels):
    """The same of the assembly with a count raised by one."""
    D, (_, on, _) = kernels
    pieces, seen = _pieces(D), 0
    name, lines = on[0]
    for i in [i for i, s in enumerate(lines) if re.search(rf"s_waitcnt vmcnt\({pieces}\)\s*$", s) and "#ASMSTART" in lines[i - 1]]:
        spoilt = list(lines)
        spoilt[i] = f"\ts_waitcnt vmcnt({pieces + 1})"
        with pytest.raises(AssertionError):
            _check_all(name, spoilt, pieces)
        seen += 1
    assert seen == 2        # for the keys, and for the values


def test_the_loop_waits_by_hand_alone(kernels):
    """No wait of the compiler's for loads in the loop over the keys, and nothing that is kept in memory."""
    for name, lines in kernels[1][0]:
        loops, where, hand = {}, None, False
        for line in lines:
            if re.match(r"\.LBB\w+:|; %bb", line):
                inside = re.search(r"in Loop: Header=(BB\w+) Depth=2", line)
                where = inside.group(1) if inside else None
                label = re.match(r"\.L(BB\w+):", line)
                own = label and label.group(1)
            if re.search(r"Inner Loop Header: Depth=2", line):
                where = own
            hand = "#ASMSTART" in line or (hand and "#ASMEND" not in line)
            if where and not line.lstrip().startswith(";"):
                loops.setdefault(where, []).append((line.strip(), hand))
        stages = [body for body in loops.values() if any("mfma" in s for s, _ in body)]
        assert len(stages) == 1 and any(INTO_LDS.match(s) for s, _ in stages[0]), (name, len(stages))
        assert not [s for s, by_hand in stages[0] if "vmcnt" in s and not by_hand], name
        assert not [s for s, _ in stages[0] if s.startswith("scratch_")], name
