"""The barriers of extend_kernel, run on the host: extend_protocol.cpp explores every interleaving of
the kernel's roles on the step order of csrc/extend_steps.h, which the kernel uses."""

import pathlib
import shutil
import subprocess

import pytest

ROOT = pathlib.Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("g++ not found")
    binary = tmp_path_factory.mktemp("protocol") / "extend_protocol"
    subprocess.run([compiler, "-O2", "-std=c++17", "-Wall", "-Werror",
                    "-I", str(ROOT / "flash-attention-lab_b200" / "csrc"),
                    str(ROOT / "tests" / "extend_protocol.cpp"), "-o", str(binary)], check=True)

    def run(*args):
        done = subprocess.run([str(binary), *args], capture_output=True, text=True, timeout=300)
        return done.returncode, done.stdout

    return run


def test_softmax_warpgroups_never_wait_for_a_phase_two_ahead(model):
    code, text = model("softmax", "joined")
    assert code == 0, text
    # The model sees the fault where only the items of one tile make the chains meet.
    code, text = model("softmax", "dual")
    assert code == 1 and "two-tile(0, 1) two-tile(0, 1)" in text and "s_full" in text


def test_scales_are_not_overwritten_while_they_are_read(model):
    code, text = model("scales", "kept")
    assert code == 0, text
    code, text = model("scales", "fewer")
    assert code == 1 and "goes on before step" in text


def test_converters_never_wait_for_a_phase_two_ahead(model):
    code, text = model("codes", "release")
    assert code == 0, text
    # A place's last tile may be the other converter's, and its copy the last to land.
    code, text = model("codes", "full")
    assert code == 1 and "3 places" in text and "code_full" in text
