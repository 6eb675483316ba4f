"""Refusals of the KV-cache operators: phase 1 is host code, so descriptors with addresses that nobody dereferences are
enough (as in test_abi_validation_cpu.py)."""
import ctypes
import os
from ctypes import POINTER, c_char_p, c_double, c_int, c_int64, c_uint64, c_void_p

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "cann-ops-adv-vllm_amd", "lib", "libcust_opapi.so")
F32, F16, I8, I32, U8, I64, BF16 = 0, 1, 2, 3, 4, 9, 27
NULLPTR, INVALID = 161001, 161002
WS = [POINTER(c_uint64), POINTER(c_void_p)]


@pytest.fixture(scope="module")
def lib():
    L = ctypes.CDLL(LIB)
    T = c_void_p
    L.aclCreateTensor.restype = T
    L.aclCreateTensor.argtypes = [POINTER(c_int64), c_uint64, c_int, POINTER(c_int64), c_int64, c_int, POINTER(c_int64), c_uint64, T]
    L.aclCreateTensorList.restype = T
    L.aclCreateTensorList.argtypes = [POINTER(T), c_uint64]
    L.aclGetRecentErrMsg.restype = c_char_p
    L.aclDestroyAclOpExecutor.argtypes = [T]
    L.aclnnAppendKvCacheGetWorkspaceSize.argtypes = [T] * 10 + [c_int64] * 4 + [T] * 5 + WS
    L.aclnnGatherKvCacheGetWorkspaceSize.argtypes = [T] * 9 + [c_int64] * 3 + [T] * 2 + WS
    L.aclnnPagedAttentionInt4GetWorkspaceSize.argtypes = [T] * 9 + [c_double] + [c_int64] * 5 + [T] * 2 + WS
    L.aclnnAssignBlockIdsGetWorkspaceSize.argtypes = [T] * 7 + [c_int64, c_int64, T] + WS
    L.aclnnPagedAttentionInt4.argtypes = [T, c_uint64, T, T]
    return L


class Desc(tuple):
    """(shape, dtype, address, strides)"""


def t(shape, dtype, addr=0x100000, strides=None):
    return Desc((tuple(shape), dtype, addr, strides))


def make(L, d):
    if d is None:
        return None
    shape, dtype, addr, strides = d
    n = len(shape)
    if strides is None:
        strides = [1] * n
        for i in range(n - 2, -1, -1):
            strides[i] = strides[i + 1] * shape[i + 1]
    dims = (c_int64 * n)(*shape)
    return L.aclCreateTensor(dims, n, dtype, (c_int64 * n)(*strides), 0, 2, dims, n, c_void_p(addr))


def plan(L, fn, args):
    ws, ex = c_uint64(0), c_void_p()
    st = fn(*[make(L, a) if isinstance(a, (Desc, type(None))) else a for a in args], ctypes.byref(ws), ctypes.byref(ex))
    if st == 0:
        L.aclDestroyAclOpExecutor(ex)
    return st, ws.value, (L.aclGetRecentErrMsg() or b"").decode()


def cache4(blocks=9, H=2, bs=32, D=64):
    return dict(kc=t((blocks, H, bs, D // 2), U8), vc=t((blocks, H, bs // 4, D // 2, 4), U8), kp=t((blocks, H, bs, 2), F16),
                vp=t((blocks, H, bs, 2), F16))


def append(L, **o):
    a = dict(key=t((5, 2, 64), F16), value=t((5, 2, 64), F16), query=t((5, 8, 64), F16, 0x200000), cs=t((100, 64), F32), positions=None,
             table=t((5, 4), I32), seq=t((5,), I32), start=None, scale=None, offset=None, bs=32, inter=0, mode=0, rest=0, **cache4(),
             out=t((5, 8, 64), F16, 0x300000))
    a.update(o)
    return plan(L, L.aclnnAppendKvCacheGetWorkspaceSize,
                [a[k] for k in ("key", "value", "query", "cs", "positions", "table", "seq", "start", "scale", "offset", "bs", "inter", "mode",
                                "rest", "kc", "vc", "kp", "vp", "out")])


def cache16(dtype=F16, shape=(9, 32, 2, 64)):
    return dict(kc=t(shape, dtype), vc=t(shape, dtype), kp=None, vp=None)


def test_append_plans(lib):
    assert append(lib)[:2] == (0, 0)
    assert append(lib, start=t((6,), I32))[0] == 0
    assert append(lib, query=None, out=None, cs=None)[0] == 0
    for shape in ((9, 32, 2, 64), (9, 2, 32, 64), (9, 32, 128)):
        assert append(lib, **cache16(F16, shape))[0] == 0
        assert append(lib, **cache16(I8, shape), scale=t((2, 2, 64), F16), offset=t((2, 2, 64), F16))[0] == 0
    assert append(lib, **cache16(I8), scale=t((2,), F16))[0] == 0
    assert append(lib, **cache16(I8), scale=t((2, 2), F16), mode=2)[0] == 0
    assert append(lib, out=t((5, 8, 64), F16, 0x200000))[0] == 0                    # in place
    assert append(lib, key=t((5, 2, 64), F16, 0x100002, (777, 65, 1)))[0] == 0      # any strides and alignment


@pytest.mark.parametrize("over,word", [
    (dict(key=None), "key"), (dict(value=t((5, 2, 32), F16)), "value"), (dict(value=t((5, 2, 64), BF16)), "value"),
    (dict(key=t((5, 2, 64), F32), value=t((5, 2, 64), F32)), "dtype"), (dict(out=None), "together"), (dict(query=None), "together"),
    (dict(key=t((5, 2, 64), F16, 0x100000, (128, 64, 2))), "contiguous"), (dict(query=t((4, 8, 64), F16)), "query"),
    (dict(out=t((5, 8, 64), F16, 0x200080)), "overlap"), (dict(out=t((5, 8, 64), F16, 0x300000, (64, 64, 1))), "overlap"),
    (dict(cs=t((100, 65), F32)), "even"), (dict(cs=t((100, 66), F32)), "head dim"), (dict(cs=t((100, 64), BF16)), "cos_sin"),
    (dict(positions=t((4,), I32)), "positions"), (dict(positions=t((5,), I64)), "positions"), (dict(cs=None, positions=t((5,), I32)), "cos_sin"),
    (dict(table=t((4, 4), I32)), "block_table"), (dict(table=t((5, 4), I64)), "block_table"), (dict(table=t((5, 0), I32)), "block_table"),
    (dict(seq=t((4,), I32)), "one"), (dict(start=t((5,), I32)), "query_start"), (dict(seq=t((0,), I32)), "sequences"),
    (dict(bs=24), "blockSize"), (dict(bs=0), "blockSize"), (dict(bs=1024), "blockSize"), (dict(table=t((5, 1 << 22), I32)), "2^26"),
    (dict(kp=None), "NULL"), (dict(kp=t((9, 2, 32, 2), F32)), "key_params"), (dict(vp=t((9, 2, 16, 2), F16)), "params"),
    (dict(kc=t((9, 2, 32, 64), U8)), "4-bit"), (dict(vc=t((9, 2, 32, 32), U8)), "4-bit"), (dict(vc=t((8, 2, 8, 32, 4), U8)), "4-bit"),
    (dict(kc=t((9, 2, 32, 32), U8, 0x100008)), "16 bytes"), (dict(scale=t((2,), F16)), "int8"),
    (dict(cache16(), kp=t((9, 2, 32, 2), F16)), "4-bit"), (dict(cache16(BF16)), "dtype"), (dict(cache16(F16, (9, 32, 3, 64))), "KV cache"),
    (dict(cache16(), vc=t((8, 32, 2, 64), F16)), "agree"), (dict(cache16(), scale=t((2,), F16)), "not int8"), (dict(cache16(I8)), "antiquantScale"),
    (dict(cache16(I8), scale=t((2, 64), F16)), "antiquantScale"), (dict(cache16(I8), scale=t((2,), F32)), "antiquantScale"),
    (dict(cache16(I8), scale=t((2,), F16), offset=t((2, 2, 64), F16)), "antiquantOffset"), (dict(cache16(I8), scale=t((2,), F16), mode=1), "mode"),
    (dict(cache16(I8, (9, 16, 2, 64)), scale=t((2,), F16), bs=16), "blockSize"),
])
def test_append_refusals(lib, over, word):
    st, _, msg = append(lib, **over)
    assert st in (NULLPTR, INVALID) and word in msg, msg


def test_head_dims(lib):
    for D in (48, 96, 16, 1024):
        assert append(lib, key=t((5, 2, D), F16), value=t((5, 2, D), F16), query=None, out=None, cs=None, **cache16(F16, (9, 32, 2, D)))[0] == INVALID
    st, _, msg = append(lib, key=t((5, 2, 512), F16), value=t((5, 2, 512), F16), query=None, out=None, cs=None, **cache4(D=512))
    assert st == INVALID and "4-bit" in msg
    assert append(lib, key=t((5, 2, 512), F16), value=t((5, 2, 512), F16), query=None, out=None, cs=None, **cache16(F16, (9, 32, 2, 512)))[0] == 0


def gather(L, **o):
    a = dict(**cache4(), table=t((5, 4), I32), seq=t((5,), I32), start=None, scale=None, offset=None, bs=32, mode=0, rest=1,
             k=t((5, 2, 64), BF16), v=t((5, 2, 64), BF16))
    a.update(o)
    return plan(L, L.aclnnGatherKvCacheGetWorkspaceSize,
                [a[k] for k in ("kc", "vc", "kp", "vp", "table", "seq", "start", "scale", "offset", "bs", "mode", "rest", "k", "v")])


def test_gather(lib):
    assert gather(lib)[:2] == (0, 0)
    for over, word in ((dict(v=t((5, 2, 64), F16)), "valueOut"), (dict(k=t((5, 2, 64), F32), v=t((5, 2, 64), F32)), "dtype"),
                       (dict(k=t((5, 2, 64), BF16, 0x100000, (256, 64, 1))), "contiguous"), (dict(k=t((5, 2, 64), BF16, 0x100004)), "16 bytes"),
                       (dict(cache16(F16)), "dtype"), (dict(kc=None), "key cache"), (dict(k=None), "keyOut"),
                       (dict(k=t((6, 2, 64), BF16), v=t((6, 2, 64), BF16)), "one")):
        st, _, msg = gather(lib, **over)
        assert st in (NULLPTR, INVALID) and word in msg, msg


def attention(L, **o):
    a = dict(q=t((5, 8, 64), F16), **cache4(), table=t((5, 4), I32), seq=t((5,), I32), start=None, lists=None, scale=0.125, H=2, bs=32, most=0,
             causal=1, rest=1, out=t((5, 8, 64), F16), lse=None)
    a.update(o)
    return plan(L, L.aclnnPagedAttentionInt4GetWorkspaceSize,
                [a[k] for k in ("q", "kc", "vc", "kp", "vp", "table", "seq", "start", "lists", "scale", "H", "bs", "most", "causal", "rest", "out", "lse")])


def test_attention_plans(lib):
    st, ws, _ = attention(lib)
    assert st == 0 and ws >= 256
    assert attention(lib, out=t((5, 8, 64), F32), lse=t((5, 8), F32))[0] == 0
    assert attention(lib, start=t((6,), I32), most=3, q=t((11, 8, 64), F16), out=t((11, 8, 64), F16))[0] == 0
    assert attention(lib, lists=t((5, 2, 7), I32))[0] == 0 and attention(lib, lists=t((6, 8, 4096), I32))[0] == 0


@pytest.mark.parametrize("over,word", [
    (dict(q=None), "query"), (dict(q=t((5, 8, 64), F32)), "query"), (dict(q=t((5, 7, 64), F16)), "divisible"), (dict(H=0), "kv heads"),
    (dict(q=t((5, 160, 64), F16), out=t((5, 160, 64), F16)), "group"), (dict(out=t((5, 8, 64), BF16)), "attentionOut"),
    (dict(out=t((5, 8, 64), F16, 0x100000, (1024, 64, 1))), "attentionOut"), (dict(out=t((4, 8, 64), F16)), "attentionOut"),
    (dict(out=t((5, 8, 64), F16, 0x100004)), "16 bytes"), (dict(out=None), "attentionOut"), (dict(lse=t((5, 7), F32)), "softmaxLse"),
    (dict(lse=t((5, 8), F16)), "softmaxLse"), (dict(scale=float("nan")), "scaleValue"), (dict(scale=float("inf")), "scaleValue"),
    (dict(start=t((6,), I32), most=0), "maxQueryLen"), (dict(start=t((6,), I32), most=1, lists=t((5, 2, 7), I32)), "block_position"),
    (dict(lists=t((5, 3, 7), I32)), "block_position"), (dict(lists=t((4, 2, 7), I32)), "block_position"), (dict(lists=t((5, 2, 5000), I32)), "4096"),
    (dict(kc=t((9, 2, 32, 64), U8)), "4-bit"), (dict(kc=t((9, 2, 32, 32), I8)), "dtype"), (dict(vp=None), "NULL"), (dict(bs=40), "blockSize"),
    (dict(seq=t((4,), I32)), "one"), (dict(table=t((5, 1 << 22), I32)), "2^26"),
])
def test_attention_refusals(lib, over, word):
    st, _, msg = attention(lib, **over)
    assert st in (NULLPTR, INVALID) and word in msg, msg


def test_wide_groups_in_lists(lib):
    big = dict(q=t((5, 128, 256), F16), out=t((5, 128, 256), F16), **cache4(D=256))
    st, _, msg = attention(lib, lists=t((5, 2, 7), I32), **big)
    assert st == 0, msg
    assert attention(lib, lists=t((5, 128, 7), I32), **big)[0] == 0


def test_assign_over_a_4_bit_cache(lib):
    def assign(kc=t((9, 2, 32, 32), U8), par=t((9, 2, 32, 2), F16), offset=None, D=64):
        keys = lib.aclCreateTensorList((c_void_p * 1)(make(lib, kc)), 1)
        ws, ex = c_uint64(0), c_void_p()
        st = lib.aclnnAssignBlockIdsGetWorkspaceSize(keys, make(lib, t((5, 4), I32)), make(lib, t((5,), I32)), make(lib, t((5,), I32)),
                                                     make(lib, t((2, 100, D), BF16)), make(lib, par), make(lib, offset), 32, 0,
                                                     make(lib, t((2, 9), I32)), ctypes.byref(ws), ctypes.byref(ex))
        if st == 0:
            lib.aclDestroyAclOpExecutor(ex)
        return st, (lib.aclGetRecentErrMsg() or b"").decode()
    assert assign()[0] == 0
    for kw, word in ((dict(par=None), "antiquantScale"), (dict(par=t((9, 2, 32, 2), BF16)), "antiquantScale"),
                     (dict(par=t((9, 2, 16, 2), F16)), "antiquantScale"), (dict(offset=t((9, 2, 32, 2), F16)), "antiquantOffset"),
                     (dict(kc=t((9, 32, 2, 32), U8)), "4-bit"), (dict(D=128), "4-bit")):
        st, msg = assign(**kw)
        assert st == INVALID and word in msg, msg


def test_phase_two_checks_the_executor(lib):
    assert lib.aclnnPagedAttentionInt4(None, 0, None, None) == NULLPTR
    ws, ex = c_uint64(0), c_void_p()
    a = [t((5, 8, 64), F16), *cache4().values(), t((5, 4), I32), t((5,), I32), None, None]
    st = lib.aclnnPagedAttentionInt4GetWorkspaceSize(*[make(lib, x) for x in a], 0.1, 2, 32, 0, 1, 1, make(lib, t((5, 8, 64), F16)), None,
                                                     ctypes.byref(ws), ctypes.byref(ex))
    assert st == 0 and ws.value > 0
    assert lib.aclnnPagedAttentionInt4(None, 0, ex, None) == INVALID          # no workspace: refused, the executor is gone


def test_python_surface_refuses_host_tensors():
    import custom_ops
    k = torch.zeros((1, 1, 64), dtype=torch.float16)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU"):
        custom_ops.append_kv_cache(k, k, k, k, i[None], i)
    with pytest.raises(RuntimeError, match="GPU"):
        custom_ops.gather_kv_cache(k, k, i[None], i, 1)
    with pytest.raises(RuntimeError, match="GPU"):
        custom_ops.paged_attention_int4(k, k, k, k, k, i[None], i, 1.0, 1)
    with pytest.raises(RuntimeError, match="head dim"):
        custom_ops.empty_int4_cache(4, 2, 16, 96, device="cpu")
    c = custom_ops.empty_int4_cache(4, 2, 32, 64, device="cpu")
    assert c.key_cache.shape == (4, 2, 32, 32) and c.value_cache.shape == (4, 2, 8, 32, 4) and c.key_params.shape == (4, 2, 32, 2)


def test_more_rows_than_a_launch_counts(lib):
    """Rows x heads of a group beyond 2^26: refused, one less is taken."""
    T = 1 << 20
    wide = dict(cache4(H=1), H=1, start=t((6,), I32), most=T)
    st, _, msg = attention(lib, q=t((T + 1, 64, 64), F16), out=t((T + 1, 64, 64), F16), **wide)
    assert st == INVALID and "2^26" in msg
    assert attention(lib, q=t((T, 64, 64), F16), out=t((T, 64, 64), F16), **wide)[0] == 0


def test_assign_counts(lib):
    """Sequences x new pages x heads beyond 2^31."""
    L = lib

    def go(B, width, most):
        keys = L.aclCreateTensorList((c_void_p * 1)(make(L, t((9, 2, 32, 32), U8))), 1)
        ws, ex = c_uint64(0), c_void_p(0)
        st = L.aclnnAssignBlockIdsGetWorkspaceSize(keys, make(L, t((B, width), I32)), make(L, t((B,), I32)), make(L, t((B,), I32)),
                                                   make(L, t((2, 100, 64), F16)), make(L, t((9, 2, 32, 2), F16)), None, 32, most,
                                                   make(L, t((2, 9), I32)), ctypes.byref(ws), ctypes.byref(ex))
        if ex.value:
            L.aclDestroyAclOpExecutor(ex)
        return st, ws.value, (L.aclGetRecentErrMsg() or b"").decode()
    st, _, msg = go(1 << 15, 1 << 15, 0)
    assert st == INVALID and "2^31" in msg
    st, ws, msg = go(1 << 15, 1 << 15, 1 << 14)
    assert st == 0 and ws > 0, msg


def test_assign_takes_a_4_bit_cache_as_the_other_operators_do(lib):
    """Its tensors start at multiples of 16 bytes."""
    def go(kc=0x100000, par=0x200000):
        keys = lib.aclCreateTensorList((c_void_p * 1)(make(lib, t((9, 2, 32, 32), U8, kc))), 1)
        ws, ex = c_uint64(0), c_void_p()
        st = lib.aclnnAssignBlockIdsGetWorkspaceSize(keys, make(lib, t((5, 4), I32)), make(lib, t((5,), I32)), make(lib, t((5,), I32)),
                                                     make(lib, t((2, 100, 64), F16)), make(lib, t((9, 2, 32, 2), F16, par)), None, 32, 0,
                                                     make(lib, t((2, 9), I32)), ctypes.byref(ws), ctypes.byref(ex))
        if st == 0:
            lib.aclDestroyAclOpExecutor(ex)
        return st, (lib.aclGetRecentErrMsg() or b"").decode()
    assert go()[0] == 0
    for kw in (dict(kc=0x100008), dict(par=0x200004)):
        st, msg = go(**kw)
        assert st == INVALID and "16 bytes" in msg, msg


def test_no_rows(lib):
    """A call without rows plans (and will launch nothing)."""
    start = t((6,), I32)
    assert append(lib, key=t((0, 2, 64), F16), value=t((0, 2, 64), F16), query=t((0, 8, 64), F16, 0x200000), out=t((0, 8, 64), F16, 0x300000),
                  start=start)[0] == 0
    assert append(lib, key=t((0, 2, 64), F16), value=t((0, 2, 64), F16), query=None, out=None, cs=None, start=start)[0] == 0
    assert gather(lib, k=t((0, 2, 64), BF16), v=t((0, 2, 64), BF16), start=start)[0] == 0
    assert attention(lib, q=t((0, 8, 64), F16), out=t((0, 8, 64), F16), start=start, most=1)[0] == 0


@pytest.mark.parametrize("addr", [0x300002, 0x300004, 0x300008])
def test_assign_over_a_4_bit_cache_needs_aligned_centroids(lib, addr):
    """The centroids go to LDS in 16-byte pieces there; a key cache of 16 bits takes them anywhere, as before."""
    def go(kc, par, cent):
        keys = lib.aclCreateTensorList((c_void_p * 1)(make(lib, kc)), 1)
        ws, ex = c_uint64(0), c_void_p()
        st = lib.aclnnAssignBlockIdsGetWorkspaceSize(keys, make(lib, t((5, 4), I32)), make(lib, t((5,), I32)), make(lib, t((5,), I32)),
                                                     make(lib, t((2, 100, 64), F16, cent)), make(lib, par), None, 32, 0,
                                                     make(lib, t((2, 9), I32)), ctypes.byref(ws), ctypes.byref(ex))
        if st == 0:
            lib.aclDestroyAclOpExecutor(ex)
        return st, (lib.aclGetRecentErrMsg() or b"").decode()
    int4 = (t((9, 2, 32, 32), U8), t((9, 2, 32, 2), F16))
    assert go(*int4, 0x300010)[0] == 0
    st, msg = go(*int4, addr)
    assert st == INVALID and "l1_cent" in msg and "16 bytes" in msg, msg
    assert go(t((9, 2, 32, 64), F16), None, addr)[0] == 0


def describe(L, fn, args):
    L.spfaDescribeExecutor.argtypes = [c_void_p, c_char_p, c_uint64]
    ws, ex = c_uint64(0), c_void_p()
    st = fn(*[make(L, a) if isinstance(a, (Desc, type(None))) else a for a in args], ctypes.byref(ws), ctypes.byref(ex))
    assert st == 0, L.aclGetRecentErrMsg()
    buf = ctypes.create_string_buffer(512)
    n = L.spfaDescribeExecutor(ex, buf, 512)
    L.aclDestroyAclOpExecutor(ex)
    assert n > 0
    return dict(part.split("=") for part in buf.value.decode().split())


@pytest.mark.parametrize("most", [1, 3, 1 << 20])
def test_a_bound_on_rows_does_not_shorten_the_arithmetic(lib, most):
    """2^20 rows over tables of 2^26 tokens may be more than 2^31 steps, whatever maxQueryLen says of them."""
    def go(T, pages):
        c = cache4(H=1)
        args = [t((T, 64, 64), F16), c["kc"], c["vc"], c["kp"], c["vp"], t((5, pages), I32), t((5,), I32), t((6,), I32), None, 0.125, 1, 32, most,
                1, 1, t((T, 64, 64), F16), None]
        return describe(lib, lib.aclnnPagedAttentionInt4GetWorkspaceSize, args)
    assert go(1 << 20, 1 << 21)["wide_line"] == "1"
    assert go(1 << 10, 1 << 10)["wide_line"] == "0"


@pytest.mark.parametrize("D,G", [(256, 33), (256, 64), (128, 64), (32, 64)])
def test_a_group_is_one_item_of_a_list(lib, D, G):
    """Lists per kv head: groups of up to 64 heads at every head dim."""
    c = cache4(H=1, D=D)
    plan = describe(lib, lib.aclnnPagedAttentionInt4GetWorkspaceSize,
                    [t((5, G, D), F16), c["kc"], c["vc"], c["kp"], c["vp"], t((5, 4), I32), t((5,), I32), None, t((5, 1, 7), I32), 0.1, 1, 32, 0, 1, 1,
                     t((5, G, D), F16), None])
    assert int(plan["rows_per_item"]) >= G and plan["lists"] == "1"


@pytest.mark.parametrize("over,word", [(dict(out_dtype=torch.bfloat16), "out_dtype"), (dict(num_tokens=4), "num_tokens"), (dict(heads=2), "heads"),
                                       (dict(heads=0), "heads"), (dict(heads=0, key_out=None, value_out=None), "heads")])
def test_gather_takes_nothing_that_its_outputs_contradict(over, word):
    import custom_ops
    k = torch.zeros((3, 1, 64), dtype=torch.float16)
    i = torch.zeros((3, 1), dtype=torch.int32)
    kw = dict(key_out=k, value_out=k.clone(), heads=1)
    kw.update(over)
    heads = kw.pop("heads")
    with pytest.raises(RuntimeError, match=word):
        custom_ops.gather_kv_cache(k[None], k[None], i, i[:, 0], heads, **kw)
    with pytest.raises(RuntimeError, match="GPU"):            # everything that agrees goes on to the next check
        custom_ops.gather_kv_cache(k[None], k[None], i, i[:, 0], 1, key_out=k, value_out=k.clone(), out_dtype=torch.float16, num_tokens=3)


def test_a_query_output_on_the_rows_it_comes_with(lib):
    """queryOut on key's or value's rows: refused.  Rows of one projection's output lie side by side without sharing anything."""
    base = 0x400000
    fused = lambda heads, at: t((5, heads, 64), F16, base + 2 * 64 * at, (12 * 64, 64, 1))       # noqa: E731   q 8, k 2, v 2 heads
    qkv = dict(query=fused(8, 0), key=fused(2, 8), value=fused(2, 10))
    assert append(lib, **qkv, out=fused(8, 0))[0] == 0
    assert append(lib, **qkv)[0] == 0
    by_head = lambda heads, at: t((5, heads, 64), F16, base + 2 * 64 * 5 * at, (64, 5 * 64, 1))   # noqa: E731
    assert append(lib, query=by_head(8, 0), key=by_head(2, 8), value=by_head(2, 10), out=by_head(8, 0))[0] == 0
    # heads apart by more than the tokens of one, tokens of the two side by side
    wide = lambda heads, at: t((5, heads, 64), F16, base + 2 * 64 * at, (2 * 64, 11 * 64, 1))      # noqa: E731
    assert append(lib, query=t((5, 8, 64), F16, 0x800000), key=wide(2, 0), value=t((5, 2, 64), F16, 0x900000), out=wide(8, 1))[0] == 0
    # heads of different widths in one token: strides differ, places in the token do not meet
    pad = lambda heads, at, head: t((5, heads, 64), F16, base + 2 * at, (2000, head, 1))         # noqa: E731
    assert append(lib, query=pad(8, 0, 80), key=pad(2, 640, 64), value=pad(2, 768, 64), out=pad(8, 0, 80))[0] == 0
    assert append(lib, query=t((5, 8, 64), F16), key=pad(2, 600, 64), value=pad(2, 768, 64), out=pad(8, 0, 80))[0] == INVALID
    one = t((5, 2, 64), F16, base + 2 * 2 * 64, (4 * 64, 64, 1))                                  # the same rows, off by half a token
    assert append(lib, query=t((5, 2, 64), F16), key=t((5, 2, 64), F16, base, (4 * 64, 64, 1)), value=t((5, 2, 64), F16, 0x700000), out=one)[0] == 0
    for over in (dict(out=t((5, 8, 64), F16, 0x500000), key=t((5, 2, 64), F16, 0x500000)),
                 dict(out=t((5, 8, 64), F16, 0x500000), value=t((5, 2, 64), F16, 0x500000 - 2 * 64)),
                 dict(qkv, query=t((5, 8, 64), F16), out=fused(8, 1)), dict(qkv, query=t((5, 8, 64), F16), out=fused(8, 3)),
                 dict(qkv, query=t((5, 8, 64), F16), out=t((5, 8, 64), F16, base))):
        st, _, msg = append(lib, **over)
        assert st == INVALID and "overlap" in msg, msg
