"""CPU: how paged decode attention divides its keys (csrc/mg_paged_plan.hpp, the
header the kernels compile) where a wave takes 32 keys at once and where it takes 64
(MXFP4 pages, heads one by one)."""
import pathlib
import subprocess

ROOT = pathlib.Path(__file__).resolve().parents[1]


def test_steps_of_32_and_64(tmp_path):
    exe = tmp_path / "paged_steps_check"
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", str(ROOT / "tests" / "host" / "paged_steps_check.cpp"),
                    "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=100)
    assert r.stdout.strip() == "ok", r.stdout
