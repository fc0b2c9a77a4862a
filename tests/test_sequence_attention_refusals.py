"""What attention between sequences refuses on the host, before anything is launched, and the map of buckets."""
import ctypes
import math

import pytest
import torch

from crystalframer_amd import _lib, cuda_funcs

A = 4096          # an address that no refused call looks at


def _args(**change):
    a = _lib.CfhAttention()
    a.struct_size, a.batch, a.heads, a.kv_heads, a.dim, a.scale, a.query_rows, a.key_rows = ctypes.sizeof(a), 2, 4, 2, 16, 0.25, 5, 7
    a.q = a.k = a.v = A
    for name, strides in (("q_stride", (320, 64, 16)), ("k_stride", (224, 32, 16)), ("v_stride", (224, 32, 16))):
        setattr(a, name, (ctypes.c_int64 * 3)(*strides))
    for k, v in change.items():
        setattr(a, k, (ctypes.c_int64 * 3)(*v) if isinstance(v, tuple) else v)
    return a


TABLE = dict(table=A, buckets=4, reach=8, bucket_of=A)


@pytest.mark.parametrize("change,word", [
    (dict(struct_size=8), b"struct_size"), (dict(dtype=3), b"dtype"), (dict(dtype=-1), b"dtype"), (dict(dim=0), b"dim"), (dict(dim=129), b"dim"),
    (dict(heads=0), b"heads"), (dict(kv_heads=3), b"heads"), (dict(kv_heads=0), b"heads"), (dict(heads=65536, kv_heads=1), b"heads"),
    (dict(batch=-1), b"batch"), (dict(query_rows=-1), b"rows"), (dict(key_rows=1 << 31), b"rows"), (dict(scale=0.0), b"scale"),
    (dict(scale=-1.0), b"scale"), (dict(scale=math.nan), b"scale"), (dict(scale=math.inf), b"scale"), (dict(q_stride=(1, -1, 1)), b"strides"),
    (dict(packed=1), b"query_starts"), (dict(packed=1, query_starts=A), b"query_starts"), (dict(query_starts=A, key_starts=A), b"packed"),
    (dict(packed=1, query_starts=A, key_starts=A, key_sizes=A), b"sizes"), (dict(q=None), b"NULL"), (dict(v=None), b"NULL"),
    (dict(k=A + 4), b"address"), (dict(dtype=1, q=A + 2), b"address"), (dict(k_stride=(224, 30, 16)), b"16 bytes"),
    (dict(v_stride=(0, 1 << 22, 16)), b"strides"), (dict(q_stride=(1 << 62, 64, 16)), b"strides"), (dict(TABLE, dtype=1, table_dtype=2), b"table_dtype"),
    (dict(TABLE, reach=1025), b"reach"), (dict(TABLE, reach=-1), b"reach"), (dict(TABLE, buckets=0), b"buckets"), (dict(TABLE, bucket_of=None), b"bucket_of"),
    (dict(buckets=3), b"table"), (dict(bucket_of=A), b"table"), (dict(TABLE, scale=2.0 ** -65), b"scale"),
    (dict(batch=0x7fffffff, key_rows=0x7fffff00), b"too many")])
def test_arguments(change, word):
    lib, a = _lib.load(), _args(**change)
    assert lib.cfh_attention_forward(ctypes.byref(a), A, None, None, A, 1 << 30, None) < 0 and word in lib.cfh_last_error()
    assert lib.cfh_attention_forward_workspace_bytes(ctypes.byref(a)) == 0
    assert lib.cfh_attention_backward_workspace_bytes(ctypes.byref(a)) == 0
    strides = (ctypes.c_int64 * 3)(320, 64, 16)
    assert lib.cfh_attention_backward(ctypes.byref(a), A, None, A, A, strides, A, A, A, None, A, 1 << 30, None) < 0 and word in lib.cfh_last_error()


@pytest.mark.parametrize("change", [dict(batch=1 << 20, query_rows=1 << 19), dict(batch=1 << 30, query_rows=1, key_rows=1)])
def test_grids(change):
    lib, a = _lib.load(), _args(heads=128, kv_heads=1, **change)
    strides = (ctypes.c_int64 * 3)(320, 64, 16)
    assert lib.cfh_attention_forward(ctypes.byref(a), A, None, None, A, 1 << 62, None) < 0 and b"grid" in lib.cfh_last_error()
    assert lib.cfh_attention_backward(ctypes.byref(a), A, None, A, A, strides, A, A, A, None, A, 1 << 62, None) < 0 and b"grid" in lib.cfh_last_error()


def test_results_and_workspaces():
    lib, a = _lib.load(), _args()
    strides = (ctypes.c_int64 * 3)(320, 64, 16)
    need = lib.cfh_attention_backward_workspace_bytes(ctypes.byref(a))
    assert need > 0

    def backward(out=A, stats=A, go=A, st=strides, dq=A, dk=A, dv=A, table=None, ws=A, n=need, args=a, rest=None):
        return lib.cfh_attention_backward(ctypes.byref(args), out, rest, stats, go, st, dq, dk, dv, table, ws, n, None)
    for change, word in ((dict(out=None), b"NULL"), (dict(stats=None), b"NULL"), (dict(go=None), b"NULL"), (dict(st=None), b"NULL"),
                         (dict(dq=None), b"NULL"), (dict(dk=None), b"together"), (dict(dv=None), b"together"), (dict(dq=A + 8), b"16"),
                         (dict(out=A + 4), b"16"), (dict(table=A), b"table"), (dict(ws=None), b"workspace"), (dict(n=need - 1), b"workspace"),
                         (dict(ws=A + 4), b"workspace"), (dict(go=A + 4), b"address"), (dict(rest=A), b"out_rest"), (dict(args=_args(dtype=1)), b"out_rest"), (dict(st=(ctypes.c_int64 * 3)(4, -4, 4)), b"strides")):
        assert backward(**change) < 0 and word in lib.cfh_last_error(), (change, lib.cfh_last_error())
    assert lib.cfh_attention_forward(ctypes.byref(a), None, None, None, None, 0, None) < 0 and b"out" in lib.cfh_last_error()
    assert lib.cfh_attention_forward(ctypes.byref(a), A + 8, None, None, None, 0, None) < 0 and b"out" in lib.cfh_last_error()
    assert lib.cfh_attention_forward(None, A, None, None, None, 0, None) < 0
    assert lib.cfh_attention_forward(ctypes.byref(a), A, A, None, None, 0, None) < 0 and b"out_rest" in lib.cfh_last_error()
    long = _args(batch=1, query_rows=1, key_rows=1 << 16)          # keys in parts
    need = lib.cfh_attention_forward_workspace_bytes(ctypes.byref(long))
    assert need > 0
    for ws, n in ((None, need), (A, need - 1), (A + 8, need)):
        assert lib.cfh_attention_forward(ctypes.byref(long), A, None, None, ws, n, None) == -2


def test_struct_matches_the_header():
    import os
    import re
    header = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "crystalframer_hip.h")).read()
    body = re.sub(r"/\*.*?\*/", "", header[header.index("typedef struct cfh_attention {"):header.index("} cfh_attention;")], flags=re.S)
    names = [re.sub(r"\[\d+\]", "", n).strip(" *") for line in re.findall(r"(?:const )?(?:int32_t|int64_t|float|void|uint8_t)\b([^;{]*);", body)
             for n in re.sub(r"const (?:void|int64_t|int32_t|uint8_t)", "", line).split(",")]
    assert names == [f[0] for f in _lib.CfhAttention._fields_]


def test_cpu_tensors():
    x = torch.zeros(1, 2, 3, 8)
    with pytest.raises(RuntimeError, match="HIP device"):
        cuda_funcs.cross_attention(x, x, x)
    with pytest.raises(RuntimeError, match="HIP device"):
        cuda_funcs.relative_attention(x, x, x, torch.zeros(4, 3), cuda_funcs.position_buckets(4, 8))
    for scale in (0.0, -1.0, math.nan):
        with pytest.raises(ValueError, match="scale"):
            cuda_funcs.cross_attention(x, x, x, scale=scale)
    with pytest.raises(ValueError, match="None"):
        cuda_funcs.relative_attention(x, x, x, None, None)


@pytest.mark.parametrize("n,distance,both", [(32, 128, True), (32, 128, False), (4, 3, True), (2, 5, False), (128, 1024, False), (47, 77, True)])
def test_buckets(n, distance, both):
    got = cuda_funcs.position_buckets(n, distance, both)
    assert got.dtype == torch.int32 and got.shape == (2 * distance + 1,)
    each = n // 2 if both else n
    e = each // 2
    for r, b in zip(range(-distance, distance + 1), got.tolist()):
        d = abs(r) if both else max(0, -r)
        first = each if both and r > 0 else 0
        if d < e:
            assert b == first + d
            continue
        x = (each - e) * math.log(d / e) / math.log(distance / e)
        assert b - first == min(each - 1, e + math.floor(x)) or (abs(x - round(x)) < 1e-9 and b - first == min(each - 1, e + round(x)))
    if both:
        assert got[0] == each - 1 and got[-1] == 2 * each - 1


@pytest.mark.parametrize("n,distance,both", [(3, 8, True), (1, 8, False), (32, 8, True), (32, 1025, True), (32, 16, False), (0, 5, True)])
def test_bucket_refusals(n, distance, both):
    with pytest.raises(ValueError, match="buckets up to distance"):
        cuda_funcs.position_buckets(n, distance, both)
