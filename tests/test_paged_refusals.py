"""What the calls for many sequences refuse, and with which words: CPU tests on a HIP runtime without a device (see test_launches.py)."""
import numpy as np
import pytest

from test_launches import launches, stub  # noqa: F401

SETUP = """
T, H, KV, D, PAGE, PAGES, SEQS = 6, 8, 2, 64, 16, 4, 2
big = space(1 << 20)
at = lambda off: big.ctypes.data + off
def v2(off=0, rows=T, cols=H * D, stride=None, inner=1):
    s = cols if stride is None else stride
    return N.TensorView2D(at(off) if off is not None else None, rows, cols, s, inner, ((rows - 1) * s + (cols - 1) * inner + 1) * 4)
def v3(off=0, d=(T, H, D), s=(H * D, D, 1)):
    return N.TensorView3D(at(off), *d, *s, (sum((n - 1) * m for n, m in zip(d, s)) + 1) * 4)
def rope(**kw):
    f = dict(dims=D, mode=2, base=10000.0, freq_scale=1.0, ext_factor=0.0, attn_factor=1.0, beta_fast=32.0, beta_slow=1.0, original_context=0, freq_factors=None)
    f.update(kw)
    return C.byref(N.Rope(*f.values()))
def cache(**kw):
    f = dict(k=at(0), v=at(0), element_type=1, num_kv_heads=KV, head_dim=D, page_size=PAGE, num_pages=PAGES, k_page_stride=PAGE * KV * D, k_token_stride=KV * D,
             k_head_stride=D, v_page_stride=PAGE * KV * D, v_token_stride=KV * D, v_head_stride=D, page_table=at(0), table_stride=4, num_seqs=SEQS, max_pages=4)
    f.update(kw)
    return C.byref(N.PagedCache(*f.values()))
P = C.c_void_p(at(0))
HALF = 1 << 19
def do_rope(result=None, input=None, positions=P, r=None):
    return L.TSHip_RoPEF32Device(result or v3(HALF), input or v3(), positions, r or rope())
def do_store(query=None, qkv=None, heads=H, c=None, starts=P, lens=P, qn=None, kn=None, r=None):
    return L.TSHip_RoPEStorePagedF32Device(query or v2(HALF), qkv or v2(cols=(H + 2 * KV) * D), heads, c or cache(), starts, lens, None, qn, kn, 1e-6, r or rope())
def do_attend(result=None, query=None, heads=H, c=None, starts=P, lens=P, scale=0.1, window=0):
    return L.TSHip_PagedAttentionF32Device(result or v2(HALF), query or v2(), heads, c or cache(), starts, lens, scale, window, None)
def do_sample(logits=None, u=P, t=P, tokens=P):
    return L.TSHip_SampleTokensF32Device(logits or v2(), u, t, None, None, None, tokens, None)
for call in calls:
    ok = eval(call)
    out.append([ok, L.TSHip_GetLastError().decode(), log()])
"""
GOOD = ["do_rope()", "do_rope(v3(), v3())", "do_rope(v3(0, s=(D, T * D, 1)), v3(HALF))", "do_rope(v3(0, s=(1024, D, 1)), v3(2048, s=(1024, D, 1)))",
        "do_rope(r=rope(ext_factor=1.0, original_context=4096, freq_scale=0.25))", "do_rope(v3(HALF, (T, H, 36), (H * 36, 36, 1)), v3(0, (T, H, 36), (H * 36, 36, 1)), r=rope(dims=8))",
        "do_store()", "do_store(v2(0, stride=(H + 2 * KV) * D))", "do_store(c=cache(element_type=0))", "do_store(c=cache(k_token_stride=D, k_head_stride=PAGE * D))", "do_attend(c=cache(k_token_stride=D))", "do_store(c=cache(element_type=30, page_size=1, num_pages=1, k_page_stride=0))",
        "do_attend()", "do_attend(v2(), v2())", "do_attend(window=5)", "do_attend(c=cache(element_type=30))", "do_attend(c=cache(element_type=0))",
        "do_attend(c=cache(num_kv_heads=1, k_head_stride=3, v_head_stride=0))", "do_attend(heads=2, query=v2(cols=2 * D), result=v2(HALF, cols=2 * D))",
        "do_sample()", "do_sample(v2(4, rows=3, cols=7, stride=9))", "do_sample(v2(0, rows=1, cols=1))"]
BAD = [
    ("do_rope(positions=None)", "positions"), ("do_rope(v3(HALF, (T, H - 1, D)))", "Size mismatch"), ("do_rope(r=rope(dims=62))", "multiple of 4"),
    ("do_rope(r=rope(dims=0))", "multiple of 4"), ("do_rope(r=rope(dims=68))", "at most head_dim"), ("do_rope(r=rope(mode=1))", "mode must be"),
    ("do_rope(r=rope(base=0.0))", "base"), ("do_rope(r=rope(base=float('nan')))", "base"), ("do_rope(r=rope(base=float('inf')))", "base"),
    ("do_rope(r=rope(freq_scale=0.0))", "freq_scale"), ("do_rope(r=rope(ext_factor=float('nan')))", "finite"), ("do_rope(r=rope(ext_factor=1.0))", "original_context"),
    ("do_rope(r=rope(ext_factor=1.0, original_context=4096, beta_fast=0.0))", "beta_fast"), ("do_rope(r=rope(ext_factor=1.0, original_context=4096, base=1.0))", "base"),
    ("do_rope(v3(HALF + 4))", "16-byte aligned"), ("do_rope(input=v3(0, s=(H * D + 2, D, 1)))", "16-byte aligned"), ("do_rope(input=v3(0, s=(2 * H * D, 2 * D, 2)))", "contiguous"),
    ("do_rope(v3(HALF, s=(D, D, 1)))", "may not overlap"), ("do_rope(v3(HALF, s=(4, H * D, 1)))", "may not overlap"), ("do_rope(v3(16), v3())", "overlaps input"),
    ("do_rope(v3(0), v3(0, s=(D, T * D, 1)))", "overlaps input"), ("do_rope(v3(HALF, (T, H, 260), (H * 260, 260, 1)), v3(0, (T, H, 260), (H * 260, 260, 1)))", "up to 256"),
    ("do_rope(v3(HALF, (T, H, 66), (H * 68, 68, 1)), v3(0, (T, H, 66), (H * 68, 68, 1)))", "multiple of 4"),
    ("do_store(heads=0)", "KV heads"), ("do_store(heads=7)", "KV heads"), ("do_store(starts=None)", "null pointer"), ("do_store(lens=None)", "null pointer"),
    ("do_store(v2(HALF, cols=H * D - 4))", "columns"), ("do_store(qkv=v2())", "columns"), ("do_store(v2(HALF, rows=T - 1))", "differ in rows"),
    ("do_store(v2(HALF, stride=H * D - 4))", "overlap"), ("do_store(v2(HALF + 8))", "16-byte aligned"), ("do_store(qn=C.c_void_p(at(4)))", "norm weights"),
    ("do_store(v2(16, stride=(H + 2 * KV) * D))", "overlaps qkv"), ("do_store(v2(0))", "overlaps qkv"), ("do_store(r=rope(dims=128))", "at most head_dim"),
    ("do_attend(c=cache(k=None))", "null pointer"), ("do_attend(c=cache(page_table=None))", "null pointer"), ("do_attend(c=cache(element_type=8))", "element type"),
    ("do_attend(c=cache(head_dim=72))", "multiple of 16"), ("do_attend(c=cache(head_dim=272))", "up to 256"), ("do_attend(c=cache(head_dim=0))", "multiple of 16"),
    ("do_attend(c=cache(num_kv_heads=3))", "KV heads"), ("do_attend(c=cache(page_size=0))", "page size"), ("do_attend(c=cache(num_pages=0))", "page size"),
    ("do_attend(c=cache(num_pages=1 << 31))", "page size"), ("do_attend(c=cache(num_seqs=0))", "page size"), ("do_attend(c=cache(max_pages=0))", "page size"),
    ("do_attend(c=cache(max_pages=1 << 28, table_stride=1 << 28))", "page size"), ("do_attend(c=cache(table_stride=3))", "page size"),
    ("do_attend(c=cache(k_token_stride=D - 8))", "strides"), ("do_attend(c=cache(v_page_stride=PAGE * KV * D + 4))", "strides"), ("do_attend(c=cache(v_head_stride=-D))", "strides"),
    ("do_attend(c=cache(v=at(8)))", "16-byte aligned"), ("do_attend(heads=4)", "columns"), ("do_attend(v2(HALF, rows=5))", "differ in rows"), ("do_attend(window=-1)", "window"),
    ("do_attend(scale=float('nan'))", "scale"), ("do_attend(scale=float('inf'))", "scale"), ("do_attend(scale=-2e38)", "scale"),
    ("do_store(c=cache(k_token_stride=D))", "overlap"), ("do_store(c=cache(v_page_stride=PAGE * KV * D - 64))", "overlap"), ("do_store(c=cache(v_head_stride=PAGE * KV * D))", "overlap"), ("do_attend(v2(16), v2())", "overlaps query"), ("do_attend(v2(None))", "Null pointer"),
    ("do_attend(query=v2(0, inner=2))", "contiguous"),
    ("do_sample(u=None)", "Invalid arguments"), ("do_sample(t=None)", "Invalid arguments"), ("do_sample(tokens=None)", "Invalid arguments"), ("do_sample(v2(0, inner=2))", "Invalid arguments"),
    ("do_sample(v2(0, rows=1, cols=(1 << 20) + 1))", "2^20"), ("do_sample(v2(None))", "Null pointer"),
]


def test_calls_that_are_served(stub):  # noqa: F811
    for call, (ok, error, log) in zip(GOOD, stub(SETUP, calls=GOOD)):
        assert ok == 1 and error == "" and launches(log, "kernel"), (call, error)


def test_calls_that_are_refused(stub):  # noqa: F811
    for (call, words), (ok, error, log) in zip(BAD, stub(SETUP, calls=[c for c, _ in BAD])):
        assert ok == 0 and words in error and not launches(log, ""), (call, error)


def test_a_launch_that_fails_is_reported(stub):  # noqa: F811
    calls = ["do_rope()", "do_store()", "do_attend()", "do_sample()"]
    got = stub(SETUP, calls=["stub.stub_fail_launch(1) or " + c for c in calls])
    for call, (ok, error, _) in zip(calls, got):
        assert ok == 0 and "stub error" in error, call


def test_the_facade_refuses_tensors_of_another_kind():
    import torch
    from tensorsharp_amd import HipBasicOps, PagedKVCache, RotaryPositions
    f, i = torch.zeros, lambda *n: torch.zeros(n, dtype=torch.int32)
    pages = f(2, 4, 1, 64)
    for k, v, table, words in [(pages[0], pages[0], i(1, 2), "4D"), (pages, pages[:1], i(1, 2), "one shape"), (pages.double(), pages.double(), i(1, 2), "Float32"),
                               (pages, pages.half(), i(1, 2), "one type"), (pages, pages, f(1, 2), "Int32"), (pages, pages, i(2), "2D"), (pages, pages, i(1, 2), "GPU memory")]:
        with pytest.raises(ValueError, match=words):
            PagedKVCache(k, v, table)
    with pytest.raises(ValueError, match="GPU memory"):
        RotaryPositions(64, freq_factors=f(32))
    with pytest.raises(ValueError, match="3D Float32"):
        HipBasicOps.RoPE(f(2, 64), f(2, 64), i(2), RotaryPositions(64))
    with pytest.raises(ValueError, match="GPU memory"):
        HipBasicOps.RoPE(f(2, 1, 64), f(2, 1, 64), i(2), RotaryPositions(64))
    with pytest.raises(ValueError, match="GPU memory"):
        HipBasicOps.SampleTokens(i(2), f(2, 64), f(2), f(2))
    with pytest.raises(ValueError, match="2D"):
        HipBasicOps.SampleTokens(i(2), f(64), f(2), f(2))


def test_the_quotient_of_a_position_by_the_page_size():
    """the multiplication that stands for it, over every kind of divisor and dividend"""
    rng = np.random.default_rng(0)
    for d in [1, 2, 3, 5, 7, 16, 24, 100, 255, 256, 4095, 4096, 65537, 2 ** 30 - 1, 2 ** 30, 2 ** 30 + 1, 2 ** 31 - 1] + [int(v) for v in rng.integers(1, 2 ** 31, 200)]:
        s = max(0, (d - 1).bit_length())
        m = ((1 << (31 + s)) + d - 1) // d
        assert m < 2 ** 32
        near = np.arange(0, 2 ** 31, max(d, 2 ** 31 // 200), dtype=np.int64)[:300]
        for n in np.concatenate([near, near - 1, near + d - 1, rng.integers(0, 2 ** 31, 200), [0, 2 ** 31 - 1]]):
            if 0 <= n < 2 ** 31:
                assert (int(n) * m) >> (31 + s) == int(n) // d, (n, d)
