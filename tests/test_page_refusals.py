"""What the calls for caches in four bits, for first positions and for the life of pages refuse, and with which words: CPU tests on a HIP runtime without
a device (see test_launches.py)."""
import pytest

from test_launches import launches, stub  # noqa: F401
from test_paged_refusals import SETUP as PAGED

SETUP = PAGED[:PAGED.index("for call in calls:")] + """
S = D // 32
def mx(**kw):
    f = dict(element_type=39, k_page_stride=PAGE * KV * D // 2, k_token_stride=KV * D // 2, k_head_stride=D // 2, v_page_stride=PAGE * KV * D // 2,
             v_token_stride=KV * D // 2, v_head_stride=D // 2)
    x = dict(k_scales=at(1 << 18), v_scales=at(3 << 17), k_scales_page_stride=PAGE * KV * S, k_scales_token_stride=KV * S, k_scales_head_stride=S,
             v_scales_page_stride=PAGE * KV * S, v_scales_token_stride=KV * S, v_scales_head_stride=S)
    for name in kw:
        (x if name in x else f)[name] = kw[name]
    f = dict(dict(k=at(0), v=at(1 << 16), num_kv_heads=KV, head_dim=D, page_size=PAGE, num_pages=PAGES, page_table=at(0), table_stride=4, num_seqs=SEQS, max_pages=4), **f)
    return C.byref(N.PagedCache(**f, **x))
def do_first(result=None, query=None, heads=H, c=None, starts=P, lens=P, scale=0.1, window=8, first=4):
    return L.TSHip_PagedAttentionFirstF32Device(result or v2(HALF), query or v2(), heads, c or cache(), starts, lens, scale, window, first, None)
def pool(**kw):
    f = dict(page_table=at(0), table_stride=4, num_seqs=SEQS, max_pages=4, page_size=PAGE, num_pages=PAGES, references=at(4096), context_lens=at(8192), scratch=at(16384))
    f.update(kw)
    return C.byref(N.PagePool(*f.values()))
def do_resize(p=None, lengths=P, moves=P, missing=P):
    return L.TSHip_ResizeSequencesDevice(p or pool(), lengths, moves, missing)
def do_fork(p=None, children=P, parents=P, count=2, moves=P, missing=P):
    return L.TSHip_ForkSequencesDevice(p or pool(), children, parents, count, moves, missing)
def do_compact(p=None, moves=P, room=3):
    return L.TSHip_CompactPagesDevice(p or pool(), moves, room)
CACHE = PAGES * PAGE * KV * D * 2
def do_copy(dst=None, src=None, moves=P, count=3):
    return L.TSHip_CopyPagesDevice(dst or cache(k=at(HALF), v=at(HALF + CACHE)), src or cache(v=at(CACHE)), moves, count)
""" + PAGED[PAGED.index("for call in calls:"):]

GOOD = ["do_store(c=mx())", "do_store(c=mx(k_token_stride=D // 2, k_head_stride=PAGE * D // 2))", "do_store(c=mx(k_scales=at(3), v_scales=at(2001)))", "do_attend(c=mx())",
        "do_attend(v2(), v2(), c=mx())", "do_attend(c=mx(k_page_stride=1 << 30, v_scales_page_stride=(1 << 32) - 1))", "do_attend(c=mx(v_page_stride=PAGE * KV * D))",
        "do_attend(c=mx(num_kv_heads=1, k_head_stride=3, v_scales_head_stride=0))", "do_attend(c=mx(), window=3)",
        "do_first()", "do_first(c=mx())", "do_first(first=0)", "do_first(window=0)", "do_first(first=(1 << 31) - 1, window=(1 << 31) - 1)", "do_first(first=(1 << 31) - 1, c=mx())",
        "do_first(v2(), v2(), c=cache(element_type=0))", "do_first(c=cache(element_type=30))",
        "do_resize()", "do_resize(pool(num_seqs=65535))", "do_resize(pool(max_pages=1 << 20, table_stride=1 << 20, page_size=1024))", "do_resize(pool(num_pages=1 << 28))",
        "do_resize(pool(num_seqs=1, table_stride=0))", "do_fork()", "do_fork(count=1)", "do_fork(count=100000)", "do_fork(pool(num_seqs=5000))", "do_compact()", "do_compact(room=1)",
        "do_compact(room=(1 << 31) - 1)", "do_copy()", "do_copy(cache(v=at(CACHE)))", "do_copy(mx(k=at(HALF), v=at(HALF + 8192), k_scales=at(HALF + 16384), v_scales=at(HALF + 20480)))",
        "do_copy(src=mx())", "do_copy(mx(), mx())", "do_copy(count=1 << 20)", "do_copy(cache(k=at(HALF), v=at(HALF + CACHE), element_type=30))",
        "do_copy(cache(k=at(HALF), v=at(HALF + CACHE), num_pages=3))", "do_copy(cache(k=at(HALF), v=at(HALF + CACHE), page_table=None, num_seqs=0, max_pages=0))"]
BAD = [
    ("do_store(c=mx(k_scales=None))", "scales of MXFP4"), ("do_attend(c=mx(v_scales=None))", "scales of MXFP4"), ("do_attend(c=mx(head_dim=48))", "multiple of 32"),
    ("do_attend(c=mx(head_dim=288))", "up to 256"), ("do_attend(c=mx(head_dim=16))", "multiple of 32"), ("do_attend(c=mx(k_token_stride=KV * D // 2 + 8))", "strides"),
    ("do_attend(c=mx(v_head_stride=16))", "strides"), ("do_attend(c=mx(k_head_stride=-D // 2))", "strides"), ("do_attend(c=mx(k=at(8)))", "16-byte aligned"),
    ("do_attend(c=mx(k_scales_head_stride=1))", "strides of the scales"), ("do_attend(c=mx(v_scales_page_stride=-64))", "strides of the scales"),
    ("do_attend(c=mx(k_scales_token_stride=0))", "strides of the scales"), ("do_attend(c=mx(k_page_stride=1 << 32))", "below 2^32"),
    ("do_attend(c=mx(v_scales_token_stride=1 << 32))", "below 2^32"), ("do_store(c=mx(k_page_stride=1 << 32))", "below 2^32"),
    ("do_store(c=mx(k_scales_token_stride=S))", "overlap"), ("do_store(c=mx(v_scales_page_stride=PAGE * KV * S - 1))", "overlap"),
    ("do_store(c=mx(v_page_stride=PAGE * KV * D // 2 - 16))", "overlap"), ("do_store(c=mx(num_kv_heads=3))", "KV heads"),
    ("do_first(first=-1)", "first"), ("do_first(window=-1)", "window"), ("do_first(starts=None)", "null pointer"), ("do_first(scale=float('nan'))", "scale"),
    ("do_first(heads=4)", "columns"), ("do_first(c=cache(k=None))", "null pointer"), ("do_first(c=mx(head_dim=48))", "multiple of 32"),
    *[("%s(pool(%s=None))" % (call, name), "null pointer") for call in ("do_resize", "do_fork", "do_compact") for name in ("page_table", "references", "context_lens", "scratch")],
    *[("%s(pool(%s))" % (call, sizes), "invalid page size") for call in ("do_resize", "do_fork", "do_compact")
      for sizes in ("num_seqs=0", "num_seqs=65536", "max_pages=0", "page_size=0", "num_pages=0", "num_pages=(1 << 28) + 1", "table_stride=3", "page_size=-16",
                    "max_pages=1 << 27, table_stride=1 << 27")],
    ("do_resize(pool(references=at(4)))", "16-byte aligned"), ("do_compact(pool(references=at(8)))", "16-byte aligned"),
    ("do_resize(lengths=None)", "null pointer"), ("do_resize(moves=None)", "null pointer"), ("do_resize(missing=None)", "null pointer"),
    ("do_fork(children=None)", "null pointer"), ("do_fork(parents=None)", "null pointer"), ("do_fork(moves=None)", "null pointer"), ("do_fork(missing=None)", "null pointer"),
    ("do_fork(count=0)", "positive"), ("do_fork(count=-1)", "positive"), ("do_compact(moves=None)", "room"), ("do_compact(room=0)", "room"), ("do_compact(room=-5)", "room"),
    ("do_copy(moves=None)", "null pointer"), ("do_copy(count=0)", "no moves"), ("do_copy(count=-3)", "no moves"),
    ("do_copy(cache(k=at(HALF), v=at(HALF + CACHE), page_size=8))", "Size mismatch"), ("do_copy(cache(k=at(HALF), v=at(HALF + CACHE), head_dim=32))", "Size mismatch"),
    ("do_copy(cache(k=at(HALF), v=at(HALF + CACHE), num_kv_heads=1))", "Size mismatch"), ("do_copy(cache(k=at(HALF), v=None))", "null pointer"),
    ("do_copy(src=cache(element_type=8))", "element type"), ("do_copy(cache(k=at(HALF), v=at(HALF + CACHE), k_token_stride=D))", "overlap"),
    ("do_copy(cache(k=at(HALF), v=at(CACHE)))", "without being the same"), ("do_copy(cache(k=at(16), v=at(CACHE + 16)))", "without being the same"),
    ("do_copy(cache(v=at(CACHE), num_pages=3))", "without being the same"), ("do_copy(cache(v=at(CACHE), element_type=30))", "without being the same"),
    ("do_copy(mx(v_scales=at((3 << 17) + 1)), mx())", "without being the same"), ("do_copy(mx(k=at(1 << 17), v=at(5 << 15), k_scales=at(7 << 16)), mx())", "without being the same"),
    ("do_copy(count=(1 << 31) - 1)", "too many pages"),
    ("do_copy(*[cache(k=at(a), v=at(a), page_size=(1 << 22) + 1, num_pages=1, k_token_stride=KV * D, v_token_stride=KV * D) for a in (0, HALF)])", "too large"),
]


def test_calls_that_are_served(stub):  # noqa: F811
    for call, (ok, error, log) in zip(GOOD, stub(SETUP, calls=GOOD)):
        assert ok == 1 and error == "" and launches(log, "kernel"), (call, error)


def test_calls_that_are_refused(stub):  # noqa: F811
    for (call, words), (ok, error, log) in zip(BAD, stub(SETUP, calls=[c for c, _ in BAD])):
        assert ok == 0 and words in error and not launches(log, ""), (call, error)


@pytest.mark.parametrize("call,kernels", [("do_store(c=mx())", 1), ("do_attend(c=mx())", 1), ("do_attend(c=mx(max_pages=4096, table_stride=4096))", 2), ("do_first()", 1), ("do_resize()", 1), ("do_resize(pool(num_pages=20000))", 3), ("do_resize(pool(num_seqs=1025))", 3), ("do_resize(pool(max_pages=20000, table_stride=20000))", 3), ("do_fork()", 1), ("do_fork(pool(max_pages=9000, table_stride=9000))", 2), ("do_fork(pool(num_seqs=5000))", 3),
                                          ("do_compact()", 1), ("do_compact(pool(num_pages=20000))", 2), ("do_copy()", 1)])
def test_a_launch_that_fails_is_reported(stub, call, kernels):  # noqa: F811
    """whichever of a call's launches it is"""
    calls = [call] + ["stub.stub_fail_launch(%d) or %s" % (i + 1, call) for i in range(kernels)]
    got = stub(SETUP, calls=calls)
    assert got[0][0] == 1 and len(launches(got[0][2], "kernel")) == kernels
    for ok, error, _ in got[1:]:
        assert ok == 0 and "stub error" in error


def test_the_scratch_of_a_pool():
    from tensorsharp_amd import hip_native as N
    size = N.lib().TSHip_PagePoolScratchDevice
    assert size(1, 1, 1) > 0 and size(65535, 1, 1 << 28) > 1 << 28 and size(100, 1000, 70000) >= 100 * 1000 + 70000
    for sizes in ((0, 1, 1), (65536, 1, 1), (1, 0, 1), (1, 1, 0), (1, 1, (1 << 28) + 1), (-1, 1, 1), (1, 1, -1)):
        assert size(*sizes) == 0


def test_the_facade_refuses_tensors_of_another_kind():
    import torch
    from tensorsharp_amd import HipBasicOps, PagedKVCache, PagePool
    i = lambda *n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    b = lambda *n: torch.zeros(n, dtype=torch.uint8)  # noqa: E731
    codes, scales, half, table = b(2, 4, 1, 32), b(2, 4, 1, 2), torch.zeros(2, 4, 1, 64).half(), i(1, 2)
    for args, words in [((codes, codes, table), "k_scales and v_scales"), ((codes, codes, table, scales), "k_scales and v_scales"), ((half, half, table, scales, scales), "only with those"),
                        ((codes, codes, table, scales.int(), scales.int()), "UInt8 scales"), ((codes, codes, table, scales, scales[:1]), "UInt8 scales"),
                        ((codes, codes, table, b(2, 4, 1, 1), b(2, 4, 1, 1)), "UInt8 scales"), ((b(2, 4, 1, 24), b(2, 4, 1, 24), table, b(2, 4, 1, 1), b(2, 4, 1, 1)), "multiple of 32"),
                        ((codes, codes, table, scales, scales), "GPU memory")]:
        with pytest.raises(ValueError, match=words):
            PagedKVCache(*args)
    for args in [(i(2), i(8), i(1), 16), (i(1, 2).long(), i(8), i(1), 16), (i(1, 2), i(8), i(1), 16)]:
        with pytest.raises(ValueError, match="2D Int32 page table in GPU memory"):
            PagePool(*args)
    for first in (-1, 2 ** 31):
        with pytest.raises(ValueError, match="first positions"):
            HipBasicOps.PagedAttention(None, None, None, None, None, 1.0, 4, first=first)
