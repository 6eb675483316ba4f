"""The device code of the KV-cache kernels as the compiler writes it: no instruction reads a matrix instruction's result before
it is there.

On gfx950 v_mfma_f32_16x16x32 needs eight wait states between the instruction and a reader of its registers that is not an
accumulating matrix instruction; the hardware does not wait by itself.  The compiler puts them in, but has been seen to miss
them across a branch (wrong cluster ids at head dim 32, and nothing else to notice it by), so the assembly of every build
configuration is searched along all paths.  Needs hipcc, no GPU."""
import os
import re
import shlex
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "cann-ops-adv-vllm_amd", "csrc")
SOURCES = ["kv_assign_int4.hip", "kv_attn_int4_f16.hip", "kv_attn_int4_bf16.hip"]
STATES = 8
# instructions without a register of their own as first operand: all operands are read
READS_ALL = ("v_cmp", "v_readlane", "v_readfirstlane", "v_fmac", "v_mac", "ds_write", "ds_max", "ds_add", "global_store", "global_atomic", "global_load_lds",
             "scratch_store", "buffer_store", "flat_store")


def registers(text):
    out = set()
    for a, b, one in re.findall(r"\bv\[(\d+):(\d+)\]|\bv(\d+)\b", text):
        out |= {int(one)} if one else set(range(int(a), int(b) + 1))
    return out


def kernels(text):
    """[(name, instructions, successors)]"""
    out, name, code, labels = [], None, [], {}
    for line in text.split("\n"):
        start = re.match(r"^(_Z\w+):", line)
        label = re.match(r"^(\.LBB\w+):", line)
        if start:
            name, code, labels = start.group(1), [], {}
        elif name and label:
            labels[label.group(1)] = len(code)
        elif name and line.startswith("\t"):
            ins = line.split(";")[0].strip()
            if ins.startswith(".end_amdhsa_kernel") or ins.startswith(".size"):
                if code:
                    out.append((name, code, labels))
                name, code = None, []
            elif ins and not ins.startswith("."):
                code.append(ins)
    done = []
    for name, code, labels in out:
        nxt = []
        for i, ins in enumerate(code):
            op, _, arg = ins.partition(" ")
            if op == "s_endpgm":
                nxt.append([])
            elif op == "s_branch":
                nxt.append([labels[arg.strip()]])
            else:
                nxt.append([i + 1] if i + 1 < len(code) else [])
                if op.startswith("s_cbranch"):
                    nxt[-1].append(labels[arg.strip()])
        done.append((name, code, nxt))
    return done


def early_readers(code, nxt):
    """(matrix instruction, reader, states between them)"""
    bad = []
    for i, ins in enumerate(code):
        if not ins.startswith("v_mfma"):
            continue
        result = registers(ins.partition(" ")[2].split(",")[0])
        todo, least = [(j, 0) for j in nxt[i]], {}
        while todo:
            j, states = todo.pop()
            if states >= STATES or least.get(j, STATES) <= states:
                continue
            least[j] = states
            op, _, args = code[j].partition(" ")
            parts = args.split(",")
            step = 1
            if op.startswith("v_mfma"):
                if registers(",".join(parts[1:3])) & result:
                    bad.append((ins, code[j], states))
                    continue
                if registers(parts[0]) & result:        # accumulates (the hardware forwards that) or starts anew
                    continue
            elif op.startswith(("v_", "ds_", "global_", "buffer_", "scratch_", "flat_")):
                read = args if op.startswith(READS_ALL) else ",".join(parts[1:])
                if registers(read) & result:
                    bad.append((ins, code[j], states))
                    continue
            elif op == "s_nop":
                step = int(args, 0) + 1
            todo += [(k, states + step) for k in nxt[j]]
    return bad


PLANTED = """
_Z4kern:
\ts_cbranch_vccz .LBB0_1
\tv_mfma_f32_16x16x32_f16 v[4:7], v[8:11], v[12:15], 0
\t{gap}
\ts_branch .LBB0_2
.LBB0_1:
\tv_mov_b32_e32 v5, 0
.LBB0_2:
\tv_cmp_gt_f32_e32 vcc, v5, v20
\ts_endpgm
\t.size _Z4kern, 4
"""


@pytest.mark.parametrize("gap,found", [("s_nop 5", 1), ("s_nop 6", 0), ("v_mfma_f32_16x16x32_f16 v[4:7], v[8:11], v[12:15], v[4:7]", 1)])
def test_the_search_finds_a_reader_behind_a_branch(gap, found):
    (_, code, nxt), = kernels(PLANTED.format(gap=gap))
    assert len(early_readers(code, nxt)) == found


@pytest.mark.skipif(shutil.which("hipcc") is None and not os.path.exists("/opt/rocm/bin/hipcc"), reason="no hipcc")
def test_no_result_is_read_early(tmp_path):
    # the compiler's command lines as the Makefile has them, to assembly instead of objects
    lines = subprocess.run(["make", "-n", "-B", "lib"], cwd=CSRC, capture_output=True, text=True, check=True).stdout.split("\n")
    jobs = []
    for src in SOURCES:
        cmd, = [shlex.split(line) for line in lines if f" {src} " in f" {line} "]
        cmd[cmd.index("-c")] = "-S"
        out = str(tmp_path / (src + ".s"))
        cmd[cmd.index("-o") + 1] = out
        jobs.append((src, out, subprocess.Popen(cmd + ["--cuda-device-only", "-Wno-everything"], cwd=CSRC)))
    for src, out, job in jobs:
        assert job.wait(timeout=900) == 0, src
        with open(out) as f:
            found = kernels(f.read())
        multiplying = [k for k in found if any(i.startswith("v_mfma") for i in k[1])]
        assert len(multiplying) >= 8, f"{src}: {len(multiplying)} kernels with matrix instructions"
        for name, code, nxt in multiplying:
            assert all(i.startswith("v_mfma_f32_16x16x32_") for i in code if i.startswith("v_mfma")), name     # (others need other waits)
            bad = early_readers(code, nxt)
            assert not bad, f"{src}, {name}: {bad[0]}"
