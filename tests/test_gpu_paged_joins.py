"""GPU: attention over pages whose keys are cut and joined, in every form of the join, and for more sequences than a wavefront has lanes.  Bounds as in
test_gpu_paged_attention.py."""
import numpy as np
import pytest

import paged_oracle as po
from paged_joins import JOINS, many
from test_gpu_paged_attention import check, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv,dim,dtype,contexts,news,window,form", JOINS)
def test_joined_pieces(hip, heads, kv, dim, dtype, contexts, news, window, form):
    import torch
    rng = np.random.default_rng(heads + dim)
    c = po.Cache(torch, rng, contexts, 16, kv, dim, getattr(torch, dtype))
    q = torch.from_numpy((2.0 * rng.standard_normal((sum(news), heads * dim))).astype(np.float32)).cuda()
    sinks = torch.from_numpy(rng.standard_normal(heads).astype(np.float32)).cuda() if heads % 2 else None
    out = run(hip, torch, c, q, news, contexts, dim ** -0.5, window, sinks)
    check(out, c, q, news, contexts, heads, dim, dim ** -0.5, window, sinks)


@pytest.mark.parametrize("group", [4, 16])
@pytest.mark.parametrize("kv", [1, 2])
def test_many_sequences_with_long_contexts(hip, kv, group):
    import torch
    rng = np.random.default_rng(kv)
    contexts, news = many(rng, kv)
    heads, dim = group * kv, 64
    c = po.Cache(torch, rng, contexts, 16, kv, dim, torch.float16)
    q = torch.from_numpy((2.0 * rng.standard_normal((sum(news) + 3, heads * dim))).astype(np.float32)).cuda()
    out = run(hip, torch, c, q, news, contexts, dim ** -0.5, rows=len(q))
    check(out[:-3], c, q[:-3], news, contexts, heads, dim, dim ** -0.5, 0, None)
    assert torch.all(out[-3:] == 7.5)
    assert torch.equal(out, run(hip, torch, c, q, news, contexts, dim ** -0.5, rows=len(q)))
