"""Who joins the parts of a row tile in the cache's attention
(csrc/kv8_join.cuh), played through on the host: whatever the order in which the
CTAs come, each row tile that several of them share is joined once, when all of
its parts are there, and all counters are zero afterwards.
"""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_every_shared_row_tile_is_joined_once(tmp_path):
    exe = tmp_path / "kv8_join_check"
    subprocess.run(["g++", "-O2", "-std=c++17", "-B/usr/lib/gcc/x86_64-linux-gnu/13/", "-I",
                    os.path.join(ROOT, "quantr-in-c_b200", "csrc"), os.path.join(ROOT, "tests", "kv8_join_check.cpp"), "-o",
                    str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.stdout.startswith("wrong 0 of "), r.stdout + r.stderr
