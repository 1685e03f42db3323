"""The check that the 4-bit cache's attentions are held to, row by row: it has to see one key too few or too many (CPU)."""
import pytest
import torch

from kv4_bounds import attention, edge_queries, worst
from test_kv4_gpu import DECODE, PREFILL, Pool


@pytest.mark.parametrize("prefill,case", [(True, c) for c in PREFILL] + [(False, c) for c in DECODE if c[4] < 5000])
def test_a_key_missing_or_too_many_is_seen(prefill, case):
    D, Hq, Hkv, T, a, window = case[:6]
    n = a + T if prefill else a
    pool = Pool(D, Hkv, [n], seed=T)
    pos = torch.arange(n - T, n)
    q = edge_queries(torch.Generator().manual_seed(T + a), pool.k[0], pos, Hq, window)
    kp = torch.arange(n)[None]
    seen = (kp <= pos[:, None]) & (kp > pos[:, None] - (window or n + 1))
    want, tol = attention(q, pool.k[0], pool.v[0], pos, window, prefill=prefill)
    assert worst(want.to(torch.bfloat16), want, tol) < 1            # (its own rounding passes)
    first = (pos - window + 1).clamp(min=0) if window else torch.zeros_like(pos)
    wrong = [(T - 1, n - 1, False), (T - 1, int(first[-1]), False)]
    if T > 1:
        wrong.append((T - 2, n - 1, True))
    if window and first[-1] > 0:
        wrong.append((T - 1, int(first[-1]) - 1, True))
    for row, key, there in wrong:
        keys = seen.clone()
        keys[row, key] = there
        if not keys[row].any():
            continue
        off, _ = attention(q[row:row + 1], pool.k[0], pool.v[0], None, keys=keys[row:row + 1], prefill=prefill)
        assert worst(off, want[row:row + 1], tol[row:row + 1]) > 2, (row, key, there)
