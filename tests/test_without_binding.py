"""custom_ops where the native binding of the KV-cache operators is not built: the other operators work as before it, the ones
that need it say so."""
import os
import subprocess
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = """
import sys
sys.path.insert(0, {pkg!r})
sys.modules["custom_ops._kv_binding"] = None          # as if the file were not there
import torch
import custom_ops
assert callable(custom_ops.sparse_paged_attention) and callable(torch.ops.myops.sparse_paged_attention)
k = torch.zeros((1, 16, 1, 64), dtype=torch.float16)
i = torch.zeros((1, 1), dtype=torch.int32)
def refused(f, error, word):
    try:
        f()
    except error as e:
        assert word in str(e), e
    else:
        raise AssertionError("not refused")
# reaches its own check of the operands (there is no GPU implementation to run here)
refused(lambda: custom_ops.assign_block_ids(k, i, i[0], k[0], i, i[0], block_size=16), RuntimeError, "GPU")
for f in (lambda: custom_ops.append_kv_cache(k[0], k[0], k, k, i, i[0]), lambda: custom_ops.gather_kv_cache(k, k, i, i[0], 1),
          lambda: custom_ops.paged_attention_int4(k[0], k, k, k, k, i, i[0], 1.0, 1),
          lambda: custom_ops.assign_block_ids(k.to(torch.uint8), i, i[0], k[0], i, i[0], block_size=16)):
    refused(f, ImportError, "make -C")
print("fine")
"""


def test_import_and_older_operators():
    r = subprocess.run([sys.executable, "-c", PROGRAM.format(pkg=os.path.join(ROOT, "cann-ops-adv-vllm_amd"))], capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr


def test_the_library_builds_by_itself():
    """`make lib` asks for nothing but the library's objects: no Python, no torch."""
    csrc = os.path.join(ROOT, "cann-ops-adv-vllm_amd", "csrc")
    out = subprocess.run(["make", "-n", "-B", "lib", "PYTHON=/nonexistent"], cwd=csrc, capture_output=True, text=True, timeout=60)
    assert out.returncode == 0 and "libcust_opapi.so" in out.stdout and "kv_binding" not in out.stdout, out.stderr
    assert "nonexistent" not in out.stderr


@pytest.mark.gpu
def test_cluster_ids_through_ctypes(monkeypatch):
    import custom_ops
    from custom_ops import _abi
    g = torch.Generator().manual_seed(1)
    dev = "cuda:0"
    key = torch.randn((20, 16, 2, 64), generator=g).half().to(dev)
    cent = torch.randn((2, 50, 64), generator=g).half().to(dev)
    table = torch.randperm(20, generator=g).view(4, 5).to(torch.int32).to(dev)
    seq = torch.tensor([80, 3, 33, 70], dtype=torch.int32, device=dev)
    got = []
    for native in (True, False):
        if not native:
            monkeypatch.setattr(_abi, "have_native", lambda: False)
        ids = torch.full((2, 20), -7, dtype=torch.int32, device=dev)
        assert custom_ops.assign_block_ids(key, table, seq, cent, ids, torch.zeros_like(seq), block_size=16) is ids
        got.append(ids)
    torch.cuda.synchronize()
    assert torch.equal(got[0], got[1]) and bool((got[0] >= 0).any())
