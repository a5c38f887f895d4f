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


def test_whole_warps_give_up_together():
    """A wait that runs out in some lanes of a warp only must not part them: every wait of a warp that goes
    on as one is followed by a vote.  Single lanes wait by themselves (the planning lane), and the
    scores are waited for without a vote, which each of the three ways on from there takes first."""
    text = KERNEL.read_text()
    body = text[text.index("chunk_attention_kernel(const MacB200ChunkArgs"):text.index("chunk_join_kernel(")]
    planner = body[body.index("warp == kPlanWarp && lane == 0"):body.index("the products of stream")]
    alone = re.findall(r"\bmbar_wait\(&ctl\.(\w+)", body)
    assert sorted(alone) == sorted(re.findall(r"\bmbar_wait\(&ctl\.(\w+)", planner) + ["s_full"])
    steps = body[body.index("mbar_wait(&ctl.s_full"):]
    steps = steps[:steps.index("mbar_arrive(&ctl.p_full[s][b]);\n        uint64_t sum")]
    ways = re.split(r"if \(h == 0 &&|if \(!any_live\)|if \(__any_sync\(0xffffffffu, grow \|\| !ok\)\)", steps)
    assert len(ways) == 4 and "break" not in ways[0] and "continue" not in ways[0]
    for way in ways[1:]:
        vote, leave = way.find("__all_sync(0xffffffffu, ok)"), re.search(r"\b(break|continue)\b", way)
        assert 0 <= vote < leave.start()
    issue = body[body.index("the products of stream"):body.index("softmax: this thread's row")]
    assert "mbar_wait" not in issue


def test_scores_wait_for_the_product_that_reads_the_weights_below_them():
    """Products of different shape and accumulator run in no promised order, so the scores of a step may be
    written over weights only once the product of those weights is done -- also for a unit's first scores,
    over the last unit's weights (the steps are counted through)."""
    text = KERNEL.read_text()
    qk = text[text.index("auto qk = [&](int i)"):]
    qk = qk[:qk.index("__syncwarp();")]
    wait, product = qk.find("warp_wait(&ctl.o_done[s][b], (t0 + i + 2) >> 1"), qk.find("mma_ss(")
    assert 0 <= wait < product and "if (!ok) return;" in qk[wait:product]
    # step n's product counts phase n / 2 of buffer n & 1; the wait of step n is for that of step n - 2,
    # and lets the first two through, before which nothing was issued
    for n in range(12):
        awaited = ((n + 2) >> 1) & 1
        before, after = (n - 2) // 2, (n - 2) // 2 + 1          # phases done without and with step n - 2
        assert (after & 1) != awaited
        assert n < 2 or (before & 1) == awaited


def test_values_are_taken_out_by_one_store_that_stands(tmp_path):
    """A block of values that two streams share: a word with an infinity or NaN goes straight to what it stays,
    for any two halves, and the kernel stores nothing in between."""
    src, exe = tmp_path / "halves.cpp", tmp_path / "halves"
    src.write_text(f"""#include <cmath>
#include <cstring>
#include "{KERNEL.parent / 'mac_b200_chunk_ring.h'}"
static bool finite(uint32_t h) {{ uint32_t b = h << 16; float f; std::memcpy(&f, &b, 4); return std::isfinite(f); }}
int main() {{
  const uint32_t other[] = {{0u, 0x3f80u, 0x7f80u, 0xff80u, 0x7fc0u, 0xffffu, 0x7f7fu, 0x0001u, 0x8000u}};
  for (uint32_t a = 0; a < 65536; ++a)
    for (uint32_t b : other)
      for (int turn = 0; turn < 2; ++turn) {{
        const uint32_t lo = turn ? b : a, hi = turn ? a : b;
        const uint32_t want = (finite(lo) ? lo : 0u) | (finite(hi) ? hi << 16 : 0u);
        const uint32_t got = mac_b200::finite_halves(lo | hi << 16);
        if (got != want || mac_b200::finite_halves(got) != got) return 1;
      }}
  return 0;
}}
""")
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", str(src), "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)]).returncode == 0
    text = KERNEL.read_text()
    out = text[text.index("if (found) {"):]
    out = out[:out.index("fence_async_smem();")]
    assert out.count("ld.shared") == 1 and out.count("st.shared") == 1 and out.count("finite_halves(w[") == 4
    assert not re.search(r"\bv\[[^\]]*\]|\*v\b|&=|\|=", out)
