"""Which values of C the MXFP4 products' tiles read and write: the address arithmetic of the kernels (skl_mx_rows.hpp) built for the host and walked
through for every number of rows, lane and pass (tests/c/mx_rows_check.cpp). What a lane loads and does not use shows in no result, so it is looked for here."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def test_every_row_that_is_read_or_written_exists(tmp_path):
    program = tmp_path / "mx_rows_check"
    subprocess.run(["g++", "-std=c++20", "-O1", "-Wall", "-Wextra", "-Werror", os.path.join(HERE, "c", "mx_rows_check.cpp"), "-o", program], check=True)
    run = subprocess.run([program], capture_output=True, text=True)
    assert run.returncode == 0 and run.stdout == "rows ok\n", run.stdout
