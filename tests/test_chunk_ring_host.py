"""CPU: the order in which the chunk attention's warps fill, use and give back its ring of K/V blocks."""
import re
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]
KERNEL = ROOT / "mac_attention_b200" / "csrc" / "mac_b200_chunk.cu"


def test_no_order_of_the_warps_fills_a_position_in_use(tmp_path):
    """Every order of the ring's model, with the shapes and the rule that the kernel is built from."""
    exe = tmp_path / "ring"
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Wextra", "-Werror",
                    str(ROOT / "tests" / "chunk_ring_model.cpp"), "-o", str(exe)], check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stdout


def test_the_kernel_fills_by_that_rule():
    text = KERNEL.read_text()
    # the groups of loading warps: the wait that they share with the model, nowhere the bare one
    groups = text[text.index("This group's positions of the unit"):text.index("own = i - n;")]
    assert "wait_to_fill(" in groups and "kv_empty" in groups
    assert not re.search(r"mbar_wait\(&ctl\.kv_empty", groups)
