"""Host side of the fused products, compiled against the library and run without a GPU: in what order
launches may overlap, and which kernel a problem runs on (fused_choice.cpp)."""
import math
import random
import shutil
import subprocess
from pathlib import Path

import pytest

from mlir_roller_b200 import _lib
import fused_shapes as shapes

HERE = Path(__file__).resolve().parent
# what a B200 answers: SMs, and the clusters of 2, 4 and 8 CTAs of these kernels that it holds at once
DEVICE = (148, 74, 33, 15)


@pytest.fixture(scope="module")
def decide(tmp_path_factory):
    """problems -> (table of kernels, one choice per problem, last line)"""
    cxx, nvcc = shutil.which("g++"), shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    include = Path(nvcc).resolve().parent.parent / "include"
    if cxx is None or not (include / "cuda.h").exists():
        pytest.skip("no C++ compiler or no CUDA headers")
    exe = tmp_path_factory.mktemp("choice") / "fused_choice"
    lib = _lib.LIB_PATH.parent
    subprocess.run([cxx, "-std=c++17", f"-I{include}", f"-I{lib / 'csrc'}", str(HERE / "fused_choice.cpp"), "-o", str(exe),
                    f"-L{lib}", "-lroller_b200", f"-Wl,-rpath,{lib}"], check=True, capture_output=True)

    def run(problems):
        text = "\n".join(" ".join(map(str, p)) for p in problems)
        lines = subprocess.run([str(exe), *map(str, DEVICE)], input=text, check=True, capture_output=True,
                               text=True).stdout.splitlines()
        kernels = [tuple(map(int, line.split()[1:])) for line in lines if line.startswith("kernel")]
        return kernels, [tuple(map(int, line.split())) for line in lines[len(kernels):-1]], lines[-1]

    return run


def test_liberties_only_behind_a_launch_that_waited(decide):
    """Each number: whether operands were read early (10), whether the wait came late (1)."""
    assert decide([])[2] == "order 0 10 1 0 1 0 1"


def covered(decide):
    problems = [p for s in shapes.BLOCK for dt in (shapes.BF16, shapes.F16) for p in shapes.block_products(*s, dt)]
    problems += [p for s in shapes.UPDATE for p in shapes.update_products(*s)]
    return set(decide(problems)[1])


def test_every_compiled_kernel_is_run_by_a_test(decide):
    compiled = {k[:4] for k in decide([])[0]}
    assert len(compiled) == 58
    assert compiled == {k[:4] for k in covered(decide)}


def test_every_choice_is_run_by_a_test(decide):
    """Whatever the rule picks for sizes all over the range, kernel and number of parts, is in the list."""
    rng = random.Random(17)

    def size(hi):
        return int(round(math.exp(rng.uniform(0.0, math.log(hi)))))

    problems = []
    for _ in range(20000):
        problems += shapes.block_products(size(20000), size(9000), size(30000), rng.choice((shapes.BF16, shapes.F16)))
        problems += shapes.update_products(rng.choice((1, 1, 2, 3, 5, 8, 16, 64)), size(9000), size(9000))
    seen = dict(zip(decide(problems)[1], problems))
    missing = {k: v for k, v in seen.items() if k not in covered(decide)}
    assert not missing
