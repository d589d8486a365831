"""CPU: how paged decode attention's partial results find their join
(csrc/mg_paged_plan.hpp, the header the kernels compile): every one joined once,
through the notes that the kernel leaves."""
import pathlib
import subprocess

ROOT = pathlib.Path(__file__).resolve().parents[1]


def test_every_partial_result_joined_once(tmp_path):
    exe = tmp_path / "paged_cut_check"
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", str(ROOT / "tests" / "host" / "paged_cut_check.cpp"),
                    "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=100).stdout.strip() == "ok"
