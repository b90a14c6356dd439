"""The plan of the chunk attention, walked through on the host (no GPU)."""

import subprocess
from pathlib import Path

HERE = Path(__file__).resolve().parent


def test_every_unit_belongs_to_one_piece(tmp_path):
    program = tmp_path / "walk"
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover",
                    str(HERE / "chunk_plan_walk.cpp"), "-o", str(program)], check=True)
    done = subprocess.run([str(program)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout == "ok\n", done.stdout + done.stderr
