"""CPU: which form of the joining kernel the calls of paged_joins.py launch, on a HIP runtime without a device (see test_launches.py)."""
import numpy as np
import pytest

from paged_joins import JOINS, many
from test_launches import launches, stub  # noqa: F401

CALL = """
a = space(64)
p = a.ctypes.data
per = 16 * kv * dim
cache = N.PagedCache(p, p, element, kv, dim, 16, 1000, per, kv * dim, dim, per, kv * dim, dim, p, width, seqs, width)
q = N.TensorView2D(p, rows, heads * dim, heads * dim, 1, rows * heads * dim * 4)
ok = L.TSHip_PagedAttentionF32Device(q, q, heads, C.byref(cache), C.c_void_p(p), C.c_void_p(p), 0.1, window, None)
out.append([ok, L.TSHip_GetLastError().decode(), log()])
"""
ELEMENT = {"float32": 0, "float16": 1, "bfloat16": 30}


def join_of(stub, heads, kv, dim, dtype, contexts, news, window):  # noqa: F811
    width = max(-(-c // 16) for c in contexts) + 1
    ((ok, error, log),) = stub(CALL, heads=heads, kv=kv, dim=dim, element=ELEMENT[dtype], rows=sum(news), seqs=len(news), width=width, window=window)
    assert ok == 1, error
    assert len(launches(log, "paged_attention_kernel")) == 1
    return [1 if "ILi1E" in l[1] else 4 for l in launches(log, "paged_combine_kernel")]


@pytest.mark.parametrize("heads,kv,dim,dtype,contexts,news,window,form", JOINS)
def test_form_of_the_join(stub, heads, kv, dim, dtype, contexts, news, window, form):  # noqa: F811
    assert join_of(stub, heads, kv, dim, dtype, contexts, news, window) == [form]


@pytest.mark.parametrize("kv", [1, 2])
def test_many_sequences_are_joined(stub, kv):  # noqa: F811
    contexts, news = many(np.random.default_rng(kv), kv)
    assert len(news) > 64 and join_of(stub, 4 * kv, kv, 64, "float16", contexts, news, 0) == [4]
    assert join_of(stub, 16 * kv, kv, 64, "float16", contexts, news, 0) == [1]
