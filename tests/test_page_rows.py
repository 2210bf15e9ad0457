"""Page plans in the middle of a step: tests/host/page_rows_test.cpp under address and undefined-behaviour sanitizers."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_page_rows_cpp(tmp_path):
    exe = str(tmp_path / "page_rows_test")
    host = os.path.join(ROOT, "warp34_amd", "host")
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-Wall", "-Wextra", "-Werror", "-fsanitize=address,undefined", "-static-libasan", "-static-libubsan",
                    os.path.join(ROOT, "tests", "host", "page_rows_test.cpp"), os.path.join(host, "kv_host.cpp"), os.path.join(host, "prefix_cache.cpp"),
                    os.path.join(host, "page_moves.cpp"), "-o", exe], check=True)
    p = subprocess.run([exe], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert p.returncode == 0, p.stdout
    assert len([l for l in p.stdout.splitlines() if l.startswith("ok ")]) == 3 and "all page row tests passed" in p.stdout, p.stdout
