"""bench.py's command line on the CPU: the one-GPU contract."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_more_than_one_gpu_exits_with_a_message():
    """--gpus above 1 ends before any GPU work with exit code 2 and says why."""
    r = subprocess.run([sys.executable, os.path.join(ROOT, "bench.py"), "--gpus", "2", "--steps", "1", "--warmup", "0"],
                       capture_output=True, text=True, timeout=60, cwd=ROOT)
    assert r.returncode == 2
    assert "one GPU only" in r.stderr
    assert r.stdout == ""


def _bench():
    if ROOT not in sys.path:
        sys.path.insert(0, ROOT)
    import bench
    return bench


def test_recorded_traffic_is_of_the_sources_in_the_tree():
    """bench.py leaves a figure out that was measured on other kernel sources: the recorded ones are of these."""
    bench = _bench()
    for workload in ("c3", "hbm1x16", "c4", "c5a", "c1", "c5gdn", "c5gdnrows"):
        assert bench.traffic_from_profiles(workload), workload


def test_recorded_traffic_depends_on_every_header_of_the_attention_kernels():
    """A header that the attention kernels include (attn_*.h) is part of their sources' hash."""
    bench = _bench()
    csrc = os.path.join(ROOT, "rust-cev_amd", "csrc")
    todo, seen = ["packed_attn.hip", "fan_attn.hip"], set()
    while todo:
        for line in open(os.path.join(csrc, todo.pop())):
            name = line.split('"')[1] if line.startswith('#include "') else ""
            if name.startswith("attn_") and name not in seen:
                seen.add(name)
                todo.append(name)
    assert seen and seen <= set(bench.K2_SOURCES)
