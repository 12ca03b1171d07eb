"""The warps of the 8-bit product kernel, played through on the CPU from the
kernel's own text: tests/f8_roles.cpp compiles the roles of csrc/f8_mm.cu as
they stand and runs every warp of a cluster in random order.

Several tiles, odd numbers of blocks, the ring of scales, both CTAs of a pair
and a shared contraction; and waits that run out, after which nothing may be
under way when a CTA ends.  A limit that runs out is not tested on a GPU:
nothing there makes one run out without a fault or a hang."""
import os
import re
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
SOURCE = os.path.join(os.path.dirname(HERE), "shoehorn_b200", "csrc", "f8_mm.cu")
SHAPES = {"128x128": 0, "128x256": 1, "pair": 2, "shared": 3, "128x128_t": 4, "128x256_t": 5, "pair_t": 6, "shared_t": 7}


def between(text, start, end):
    assert text.count(start) == 1, start
    i = text.index(start)
    return text[i:text.index(end, i)]


def build(folder, text):
    """The player of a kernel's text."""
    parts = {
        "structs": between(text, "constexpr int kTileM", "// ---------------------------------------------------------------- waits"),
        "desc": between(text, "__device__ __forceinline__ uint64_t smem_desc", "template <int PAIR>\n__device__ __forceinline__ void mma_f8"),
        "scales": between(text, "__device__ __forceinline__ void look(", "// ---------------------------------------------------------------- kernel"),
        "init": between(text, "    if (threadIdx.x == 0) {\n        for (int s = 0; s < S::kStages; s++) {", "    if (warp == S::kEpiWarps) {"),
        "roles": between(text, "    if (warp >= S::kEpiWarps) {\n        asm volatile(\"setmaxnreg", "    __syncwarp();\n    if (SPLIT) {"),
    }
    for name, part in parts.items():
        part = re.sub(r"asm volatile\(\"(setmaxnreg|fence\.mbarrier_init)[^\n]*\n", "\n", part)
        assert "asm" not in part
        (folder / f"{name}.inc").write_text(part)
    exe = str(folder / "roles")
    subprocess.run(["g++", "-std=c++17", "-O1", "-w", "-I", str(folder), "-o", exe, os.path.join(HERE, "f8_roles.cpp")], check=True)
    return exe


def play(exe, shape, seeds, fault):
    """What the runs of `seeds` print."""
    def one(seed):
        r = subprocess.run([exe, str(SHAPES[shape]), str(seed), str(int(fault))], capture_output=True, text=True, timeout=120)
        return r.stdout.strip() or f"exit status {r.returncode}"
    with ThreadPoolExecutor(4) as pool:
        return list(pool.map(one, seeds))


@pytest.fixture(scope="module")
def text():
    return open(SOURCE).read()


@pytest.fixture(scope="module")
def exe(tmp_path_factory, text):
    return build(tmp_path_factory.mktemp("roles"), text)


@pytest.mark.parametrize("shape", SHAPES)
def test_every_tile_is_summed_and_stored(exe, shape):
    assert set(play(exe, shape, range(60), False)) == {"done"}


@pytest.mark.parametrize("shape", SHAPES)
def test_a_wait_that_runs_out_leaves_nothing_under_way(exe, shape):
    said = play(exe, shape, range(150), True)
    assert set(said) <= {"done", "gave up"}
    assert said.count("gave up") > 50


EMPTY = "ok = bar_wait(&ctl.acc[h][buf].empty, acc_phase, abort, p.status);"
FULL = "if (h == 0) ok = ok && bar_wait(&ctl.full[s], phase, abort, p.status);"
MISTAKES = {  # what is put in a kernel's text, and a shape and a kind of run that show it
    "the stage awaited before the accumulator": ([(EMPTY, "ok = h != 0 || bar_wait(&ctl.full[s], phase, abort, p.status);"),
                                                  (FULL, "ok = ok && bar_wait(&ctl.acc[h][buf].empty, acc_phase, abort, p.status);")],
                                                 "128x256", False),
    "odd blocks not carried over tiles": ([("first = (first + blocks) & 1;", "")], "128x128", False),
    "one arrival too few hands an accumulator back": ([("mbar_init(&ctl.acc[h][i].empty, S::kEpiWarps / S::kHalves * PAIR)",
                                                        "mbar_init(&ctl.acc[h][i].empty, S::kEpiWarps / S::kHalves * PAIR - 1)")],
                                                      "pair", False),
    "scales written without their slot's being empty": ([("mbar_init(&ctl.slot_empty[i], S::kEpiWarps)",
                                                          "mbar_init(&ctl.slot_empty[i], 1)")], "128x256", False),
    "the last products not waited for": ([("if (rank == 0 && elect_one()) {  // its products end", "if (false) {  //")], "shared", True),
    "a pair's loading threads that do not catch up": ([("if (it < other) {", "if (false) {")], "pair", True),
    "copies not waited for": ([("wait_drain(&ctl.full[k % S::kStages], (k / S::kStages) & 1);", "break;")], "128x128", True),
}


@pytest.mark.parametrize("mistake", MISTAKES)
def test_mistakes_are_noticed(tmp_path, text, mistake):
    changes, shape, fault = MISTAKES[mistake]
    for old, new in changes:
        assert text.count(old) == 1, old
        text = text.replace(old, new)
    exe = build(tmp_path, text)
    assert any(not set(play(exe, shape, range(first, first + 12), fault)) <= {"done", "gave up"} for first in range(0, 300, 12))
