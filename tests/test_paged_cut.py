"""CPU checks of csrc/paged_cut.h, by which kernels find pages and cut the work of attention over them."""

import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "quasi-linear-kernel-attention_amd",
                    "csrc")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

# Sequences of up to a quarter of a million rows over up to 2^27 positions, whose products no float holds.
SPANS = r"""
#include "paged_cut.h"
#include <cstdio>
#include <random>
using namespace qlka::pg;
int main() {
    std::mt19937 rng(1);
    const auto upto = [&](int n) { return (int)(rng() % (unsigned)n); };
    for (int i = 0; i < 20000; ++i) {
        Extent h[9];
        const int n = 1 + upto(9), align = 128, least = i % 2 ? 128 : 256;
        const float aim = 1 + upto(1024);
        float work = 0.f;
        long long blocks = 0, units = 0;
        for (int j = 0; j < n; ++j) {
            h[j] = {upto(2 << upto(14)), upto(2 << upto(27))};
            work = more_work(work, h[j]);
            blocks += h[j].blocks;
        }
        const int span = span_of(work, aim, least, align);
        if (span % align || span < least) return 1;
        for (int j = 0; j < n; ++j) {
            const Cut c = cut_of(h[j], span, align);
            if (c.parts < 1 || c.span > span || c.span % align) return 2;
            if ((long long)c.parts * c.span < h[j].seen) return 3;             // all positions in some part
            units += (long long)c.blocks * c.parts;
        }
        if (units > blocks + (long long)aim + 1) return 4;                       // the workspace has room for so many
        std::printf("%d\n", span);
    }
    return 0;
}
"""


def run(tmp_path, source, name, *flags):
    src, exe = tmp_path / f"{name}.hip", tmp_path / name
    src.write_text(source)
    subprocess.run([HIPCC, "--offload-host-only", "-std=c++17", "-O2", *flags, f"-I{CSRC}", str(src), "-o", str(exe)],
                   check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout + done.stderr
    return done.stdout.split()


def test_spans_do_not_go_by_what_the_compiler_fuses(tmp_path):
    """The kernel that joins parts reads where another one wrote them: both find the span by themselves."""
    apart = run(tmp_path, SPANS, "apart", "-mfma", "-ffp-contract=off")
    fused = run(tmp_path, SPANS, "fused", "-mfma", "-ffp-contract=fast")
    assert len(apart) == 20000 and apart == fused
