"""CPU: how paged decode attention divides its keys (csrc/mg_paged_plan.hpp, the
header the kernels compile): every unit once, partial results in places of their
own, the join over exactly the teams that leave one."""
import pathlib
import subprocess

ROOT = pathlib.Path(__file__).resolve().parents[1]


def test_every_key_once(tmp_path):
    exe = tmp_path / "paged_plan_check"
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", str(ROOT / "tests" / "host" / "paged_plan_check.cpp"),
                    "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=100).stdout.strip() == "ok"
