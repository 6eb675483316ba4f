"""Inline assembly of the kernels names the special registers that it writes."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cann-ops-adv-vllm_amd", "csrc")


def test_m0_is_named_where_it_is_written():
    seen = 0
    for path in sorted(glob.glob(os.path.join(CSRC, "*.inc")) + glob.glob(os.path.join(CSRC, "*.hip"))):
        with open(path) as f:
            text = f.read()
        for asm in re.findall(r"\basm\s+volatile\s*\((.*?)\);", text, re.S):
            if re.search(r"\bs_\w+ m0\b", asm):
                seen += 1
                assert re.search(r':[^:]*"m0"[^:]*$', asm), f"{os.path.basename(path)}: {asm}"
    assert seen >= 7
