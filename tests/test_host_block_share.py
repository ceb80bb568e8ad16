"""Who brings what of a block of keys and values to the tiles of attention over a paged cache, on the host, without a GPU."""
import os
import subprocess

from test_host_runtime import HERE, ROOT


def test_every_piece_once_and_no_hole_without_a_key(tmp_path):
    """Each 16 bytes of each row come once, and only threads that have a row report that its key has no page: a block that is said to have holes costs every row of it the mask."""
    exe = str(tmp_path / "share")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I" + os.path.join(ROOT, "axiom_amd", "csrc", "hip"), os.path.join(HERE, "block_share_driver.cpp"), "-o", exe], check=True)
    lines = subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split("\n")[:-1]
    assert len(lines) == 12
    for line in lines:
        assert " ok, " in line and line.endswith("256 idle" if line.startswith("32 4 ") else " 0 idle"), line
