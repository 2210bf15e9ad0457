"""The scored decode kernels read no entry of a block table but those of the pages that their keys lie in: their walk, cut out of the
sources, runs on the CPU over page sizes, first half units and lengths (tests/host/page_walk_test.cpp)."""
import os
import re
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "warp34_amd", "csrc")


def cut(name, pattern):
    with open(os.path.join(CSRC, name)) as f:
        found = re.findall(pattern, f.read(), re.M | re.S)
    assert len(found) == 1, (name, pattern, len(found))
    return found[0]


def test_walk_reads_the_entries_of_its_keys_pages_only(tmp_path):
    walk = cut("scored_decode.h", r"^struct PageWalk \{.*?^\};")
    walk = re.sub(r"^.*asm volatile.*$", "", walk, flags=re.M)
    walk = walk.replace("blocks[slot + lane]", "0")  # (what a lane holds is looked at where it is read)
    parts = {
        "page_slot.inc": cut("scored_attn.h", r"^__device__ __forceinline__ int page_slot\(.*?^\}"),
        "page_walk.inc": walk,
        "tq4_locate.inc": cut("scored_decode_tq4.h", r"^    const auto locate = .*?^    \};"),
        "tq4_next.inc": cut("scored_decode_tq4.h", r"^    while \(half < end\) \{.*?\n( *[^\n]*locate\([^\n]*)"),
    }
    for name, text in parts.items():
        (tmp_path / name).write_text(text + "\n")
    exe = str(tmp_path / "page_walk_test")
    subprocess.run(["g++", "-std=c++17", "-O2", "-I", str(tmp_path), "-o", exe, os.path.join(ROOT, "tests", "host", "page_walk_test.cpp")], check=True)
    p = subprocess.run([exe], stdout=subprocess.PIPE, text=True)
    assert p.returncode == 0, p.stdout
