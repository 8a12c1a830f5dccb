"""CPU: caches whose sizes or strides multiply to more than 64 bits are refused by what copies pages or stores into them, on a HIP runtime without a
device (see test_launches.py); a division by a size that wrapped to 0 would end the process."""
from test_launches import launches, stub  # noqa: F401
from test_page_refusals import SETUP

BIG = "page_size=1 << 30, num_kv_heads=1 << 28, head_dim=256, num_pages=1, k_token_stride=1 << 36, k_head_stride=256, v_token_stride=1 << 36, v_head_stride=256"
BAD = [
    ("do_copy(*[cache(%s)] * 2)" % BIG, "too large"),
    ("do_copy(*[cache(%s)] * 2)" % BIG.replace("1 << 28", "(1 << 28) + 1").replace("1 << 36", "1 << 37"), "too large"),
    ("do_copy(*[cache(page_size=1 << 22, num_kv_heads=3, num_pages=1, head_dim=64, k_token_stride=192, v_token_stride=192)] * 2)", "too large"),
    ("do_copy(cache(k_token_stride=1 << 62, k_page_stride=(1 << 62) + D, k=at(HALF), v=at(HALF + CACHE)))", "overlap"),
    ("do_copy(*[mx(v_scales_token_stride=(1 << 32) - 1, v_scales_page_stride=(1 << 32) - 1)] * 2)", "overlap"),
    ("do_store(c=cache(k_token_stride=1 << 62, k_page_stride=(1 << 62) + D))", "overlap"),
    ("do_copy(cache(k=at(HALF), v=at(HALF + CACHE)), cache(v=at(CACHE), k_page_stride=3 << 60, num_pages=7))", "without being the same"),
    ("do_copy(cache(k=at(HALF), v=at(HALF + CACHE)), cache(v=at(CACHE), element_type=0, k_page_stride=1 << 60, num_pages=5))", "without being the same"),
]
GOOD = ["do_copy(*[cache(page_size=1 << 22, num_kv_heads=2, num_pages=1, head_dim=64)] * 2, count=1)"]


def test_sizes_beyond_64_bits(stub):  # noqa: F811
    for call, words in BAD:
        (ok, error, log), = stub(SETUP, calls=[call])
        assert ok == 0 and words in error and not launches(log, ""), (call, error)


def test_the_largest_page(stub):  # noqa: F811
    for call, (ok, error, log) in zip(GOOD, stub(SETUP, calls=GOOD)):
        assert ok == 1 and launches(log, "copy_pages"), (call, error)
