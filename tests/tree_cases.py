"""Trees of drafted tokens for the tests: parents, depths and ancestor words."""
import numpy as np
import torch


def tree(rng, n, kind="mixed"):
    """Parents, depths and which nodes lie on each node's path (itself among them) of a tree of n nodes."""
    parents, depth, on = [-1] * n, [0] * n, np.eye(n, dtype=bool)
    for i in range(1, n):
        p = {"chain": i - 1, "star": 0}.get(kind, i - 1 if rng.random() < 0.4 else int(rng.integers(0, i)))
        parents[i], depth[i] = p, depth[p] + 1
        on[i] |= on[p]
    return parents, depth, on


def words_of(on, words):
    """Truth values [n, m] as int32 words, lowest bit first."""
    n, m = on.shape
    out = np.zeros((n, words), dtype=np.uint32)
    for j in range(m):
        out[:, j // 32] |= on[:, j].astype(np.uint32) << np.uint32(j % 32)
    return torch.from_numpy(out.view(np.int32))
