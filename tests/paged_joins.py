"""Calls of the attention over pages whose keys are cut and joined, in every form of the kernel that joins: shared by the test of what is launched (CPU)
and that of the results (GPU).

JOINS: heads, kv heads, dim, type, contexts, new tokens, window, which form (1: many rows, a wavefront per row and KV head; 4: a workgroup per row and head)."""

JOINS = [
    (14, 2, 64, "float16", [2500], [170], 0, 1), (10, 2, 80, "bfloat16", [3100, 40], [230, 9], 0, 1), (6, 2, 256, "float16", [2100], [360], 0, 1),
    (6, 2, 128, "float32", [2000, 1500], [200, 170], 0, 1), (5, 1, 48, "float16", [4000], [430], 1800, 1), (7, 1, 192, "bfloat16", [2300], [310], 0, 1),
    (40, 8, 16, "float16", [4000], [70], 0, 1), (33, 3, 96, "float32", [2700], [80], 0, 1),
    (14, 2, 64, "float16", [2500], [100], 0, 4), (10, 2, 80, "bfloat16", [3100], [1], 0, 4), (6, 2, 256, "float32", [2100, 2600], [1, 3], 0, 4),
    (3, 3, 16, "float16", [6000], [40], 0, 4), (7, 1, 192, "float16", [5000, 300], [5, 1], 3000, 4), (33, 3, 128, "bfloat16", [2700], [9], 0, 4),
]


def many(rng, kv):
    """more sequences than a wavefront has lanes: answers with long and short contexts, prompts and sequences without new tokens among them; for one
    and two KV heads few enough tiles to be cut"""
    seqs = 150 if kv == 1 else 90
    contexts = [int(v) for v in rng.integers(1, 200, seqs)]
    news = [1 if v < 0.7 else 0 for v in rng.random(seqs)]
    for s, (ctx, n) in {3: (2600, 1), 17: (2300, 3), 63: (3500, 1), 64: (2900, 60), 65: (2048, 0), 70: (4000, 1), 80: (2200, 2), seqs - 1: (3100, 1)}.items():
        contexts[s], news[s] = ctx, n
    news = [min(n, c) for n, c in zip(news, contexts)]
    return contexts, news
