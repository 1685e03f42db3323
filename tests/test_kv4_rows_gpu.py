"""Attention over the 4-bit cache, every row, head and group of channels by itself: borders of the mask, and values, keys and queries of any size
(needs a B200)."""
import math

import pytest
import torch

from kv4_bounds import attention, edge_queries, worst
from r4dx_b200.quant import kv4
from test_kv4_gpu import DECODE, PREFILL, Pool, rows

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(scope="module")
def K():
    from r4dx_b200.ops import kernels
    return kernels


class Filled:
    """A pool of one sequence of given rows (bf16 [n, Hkv, D]); ``free`` is the byte of everything that no row owns."""

    def __init__(self, k, v, free=0xFF, first=0):
        n, Hkv, D = k.shape
        blocks = (n + 15) // 16
        self.table = torch.randperm(blocks + 1, generator=torch.Generator().manual_seed(n)).to(torch.int32)
        self.cache = torch.full(kv4.pool_shape(blocks + 1, Hkv, D), free, dtype=torch.uint8)
        pos = torch.arange(first, n)
        kv4.write_rows(self.cache, k[first:], v[first:], self.table[pos // 16], pos % 16)
        self.k, self.v = kv4.round_trip(k).double(), kv4.round_trip(v).double()


def decode(K, pool, q, pos, window=0, gate=None, splits=None):
    T, Hq, D = q.shape
    out = torch.full((T, Hq, D), float("nan"), dtype=BF, device="cuda")
    K.attn_decode_kv4(q.cuda(), None if gate is None else gate.cuda(), pool.cache.cuda(), pool.table.cuda(), pos.int().cuda(), out, T, Hq, pool.k.shape[1], D,
                      gate is not None, window, splits=splits)
    K.check_gemm_status(out.device)
    return out


def prefill(K, pool, q, pos0, window=0, gate=None, splits=1):
    T, Hq, D = q.shape
    out = torch.full((T, Hq, D), float("nan"), dtype=BF, device="cuda")
    K.attn_prefill_kv4(q.cuda(), None if gate is None else gate.cuda(), pool.cache.cuda(), pool.table.cuda(), out, T, Hq, pool.k.shape[1], D, pos0,
                       gate is not None, window, splits=splits)
    K.check_gemm_status(out.device)
    return out


def hold(K, k, v, q, pos, window=0, which="both"):
    """Both kernels' rows over the cache of k and v: the decode kernel by one CTA and by several, the prefill kernel (consecutive positions) alike."""
    pool = Filled(k, v)
    got = {}
    if which != "prefill":
        want, tol = attention(q, pool.k, pool.v, pos, window)
        for splits in (None, 1, 3):
            got["decode", splits] = worst(decode(K, pool, q, pos, window, splits=splits), want, tol)
    if which != "decode":
        want, tol = attention(q, pool.k, pool.v, pos, window, prefill=True)
        for splits in (1, 2):
            got["prefill", splits] = worst(prefill(K, pool, q, int(pos[0]), window, splits=splits), want, tol)
    assert max(got.values()) <= 1, got


# ---- borders of what a row sees ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("case", DECODE)
def test_decode_rows(K, case):
    D, Hq, Hkv, T, ctx, window, gated, splits = case
    g = torch.Generator().manual_seed(ctx + T)
    pool, pos = Pool(D, Hkv, [ctx], seed=ctx), torch.arange(ctx - T, ctx)
    pool.k, pool.v, pool.table = pool.k[0], pool.v[0], pool.tables[0]
    q = edge_queries(g, pool.k, pos, Hq, window)
    gate = torch.randn(T, Hq, 2 * D, generator=g).to(BF) if gated else None
    want, tol = attention(q, pool.k, pool.v, pos, window, gate=gate[..., D:] if gated else None)
    assert worst(decode(K, pool, q, pos, window, gate, splits), want, tol) <= 1


@pytest.mark.parametrize("case", PREFILL)
def test_prefill_rows(K, case):
    D, Hq, Hkv, T, pos0, window, gated, splits = case
    g = torch.Generator().manual_seed(T + pos0)
    pool, pos = Pool(D, Hkv, [pos0 + T], seed=T), torch.arange(pos0, pos0 + T)
    pool.k, pool.v, pool.table = pool.k[0], pool.v[0], pool.tables[0]
    q = edge_queries(g, pool.k, pos, Hq, window)
    gate = torch.randn(T, Hq, 2 * D, generator=g).to(BF) if gated else None
    want, tol = attention(q, pool.k, pool.v, pos, window, gate=gate[..., D:] if gated else None, prefill=splits is not None or T > 32)
    assert worst(prefill(K, pool, q, pos0, window, gate, splits), want, tol) <= 1


@pytest.mark.parametrize("D,Hq,Hkv,window", [(256, 24, 4, 0), (128, 8, 2, 40), (64, 32, 8, 0)])
def test_batch_rows(K, D, Hq, Hkv, window):
    lengths = [1, 700, 16, 33, 129, 300, 17, 1000]
    pool, g = Pool(D, Hkv, lengths, seed=5), torch.Generator().manual_seed(D)
    slot = torch.randperm(len(lengths), generator=g)
    pos = torch.tensor(lengths)[slot] - 1
    q = torch.cat([edge_queries(g, pool.k[s], p[None], Hq, window) for s, p in zip(slot.tolist(), pos)])
    out = torch.full((len(lengths), Hq, D), float("nan"), dtype=BF, device="cuda")
    K.attn_decode_kv4(q.cuda(), None, pool.cache.cuda(), pool.tables.cuda(), pos.int().cuda(), out, len(lengths), Hq, Hkv, D, False, window,
                      row_slot=slot.int().cuda())
    K.check_gemm_status(out.device)
    for b, s in enumerate(slot.tolist()):
        want, tol = attention(q[b:b + 1], pool.k[s], pool.v[s], pos[b:b + 1], window)
        assert worst(out[b:b + 1], want, tol) <= 1, s


# ---- values of any size -----------------------------------------------------------------------------------------------------------
def inputs(D, n, T, Hq, Hkv, seed):
    g = torch.Generator().manual_seed(seed)
    return rows(g, n, Hkv, D), rows(g, n, Hkv, D), torch.randn(T, Hq, D, generator=g).to(BF), torch.arange(n - T, n)


VALUES = [(256, 3.0e-5), (64, 1e-6), (128, 1e-7), (256, 1e-20), (128, 1e-35), (64, 4000.0)]


@pytest.mark.parametrize("D,size", VALUES)
def test_prefill_of_values_of_any_size(K, D, size):
    k, v, q, pos = inputs(D, 300, 40, 4, 2, D)
    hold(K, k, (v.float() * size).to(BF), q, pos, which="prefill")
    hold(K, k, (v.float() * size).to(BF), q, pos, window=50, which="prefill")


@pytest.mark.parametrize("D,size", VALUES)
def test_decode_of_values_of_any_size(K, D, size):
    k, v, q, pos = inputs(D, 300, 8, 4, 2, D)
    hold(K, k, (v.float() * size).to(BF), q, pos, which="decode")


def uneven(D, which, ratio):
    k, v, q, pos = inputs(D, 700, 8 if which == "decode" else 40, 4, 2, D)
    v = v.float()
    v[:, 0, :64] *= ratio                                   # a group against the others of its head
    v[:, 1, -64:] /= ratio
    return k, v.to(BF), q, pos


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("ratio", [2.0 ** 14, 2.0 ** 20, 2.0 ** -20])
def test_prefill_of_value_groups_far_apart(K, D, ratio):
    hold(K, *uneven(D, "prefill", ratio / 1024), which="prefill")


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("ratio", [2.0 ** 14, 2.0 ** 20, 2.0 ** -20])
def test_decode_of_value_groups_far_apart(K, D, ratio):
    hold(K, *uneven(D, "decode", ratio / 1024), which="decode")


def loud(D, T, at, groups, ratio, size=1 / 64):
    """Tokens `at` with values `ratio` times the others' (in the first `groups` channels) that no row gives a weight to speak of."""
    g = torch.Generator().manual_seed(D + T)
    Hq, Hkv, n = 4, 2, 1500
    q = (1 + 0.25 * torch.randn(T, Hq, D, generator=g)).to(BF)
    k, v = (0.1 * torch.randn(n, Hkv, D, generator=g)).to(BF), (torch.randn(n, Hkv, D, generator=g) * size).to(BF)
    for t in at:
        k[t] = -8.0
        v[t, :, :groups] = (v[t, :, :groups].float() * ratio).to(BF)
    return k, v, q, torch.arange(n - T, n)


LOUD = [(D, groups, at) for D, groups in ((64, 64), (128, 128), (128, 64), (256, 256), (256, 64)) for at in ((0,), (5, 700, 1490))]


@pytest.mark.parametrize("D,groups,at", LOUD)
def test_prefill_of_loud_tokens_without_weight(K, D, groups, at):
    hold(K, *loud(D, 40, at, groups, 2.0 ** 20), which="prefill")
    hold(K, *loud(D, 40, at, groups, 2.0 ** 20, 1e-6), which="prefill")


@pytest.mark.parametrize("D,groups,at", LOUD)
def test_decode_of_loud_tokens_without_weight(K, D, groups, at):
    hold(K, *loud(D, 8, at, groups, 2.0 ** 20), which="decode")
    hold(K, *loud(D, 8, at, groups, 2.0 ** 20, 1e-6), which="decode")


@pytest.mark.parametrize("D", [64, 128, 256])
def test_loud_tokens_whose_weight_fades(K, D):
    """The first token has a row's whole weight until others, 2^20 quieter, are met whose scores lie far above it (and again)."""
    g = torch.Generator().manual_seed(D)
    Hq, Hkv, n = 4, 2, 3000
    q = (1 + 0.25 * torch.randn(1, Hq, D, generator=g)).to(BF)
    k, v = (0.1 * torch.randn(n, Hkv, D, generator=g)).to(BF), (torch.randn(n, Hkv, D, generator=g) / 64).to(BF)
    k[:1000], k[1000:2000] = (k[:1000].float() - 10).to(BF), (k[1000:2000].float() - 5).to(BF)
    v[:1000], v[1000:2000] = (v[:1000].float() * 2.0 ** 20).to(BF), (v[1000:2000].float() * 2.0 ** 10).to(BF)
    hold(K, k, v, q, torch.tensor([n - 1]))


# ---- queries and keys of any size ---------------------------------------------------------------------------------------------------
SIZES = [(64, 1e-5, 1e4), (128, 1e-7, 2e4), (256, 2e-6, 1.6e4), (128, 3e6, 1e-6), (256, 1e20, 1e-20), (64, 1e30, 3e-31)]
LARGE = [(64, 1e7, 1e-4), (128, 1e5, 0.01), (256, 1e6, 1e-3), (64, 1e7, 1.0), (128, 1e-20, 1e4)]


@pytest.mark.parametrize("D,q_size,k_size", SIZES + LARGE)
def test_decode_of_queries_and_keys_of_any_size(K, D, q_size, k_size):
    k, v, q, pos = inputs(D, 300, 8, 4, 2, D)
    hold(K, (k.float().clamp(-2, 2) * k_size).to(BF), v, (q.float() * q_size).to(BF), pos, which="decode")


@pytest.mark.parametrize("D,q_size,k_size", LARGE)
def test_prefill_of_queries_of_any_size(K, D, q_size, k_size):
    k, v, q, pos = inputs(D, 300, 40, 4, 2, D)
    hold(K, (k.float().clamp(-2, 2) * k_size).to(BF), v, (q.float() * q_size).to(BF), pos, which="prefill")


@pytest.mark.parametrize("D,q_size,k_size", SIZES)
def test_prefill_of_queries_and_keys_of_any_size(K, D, q_size, k_size):
    k, v, q, pos = inputs(D, 300, 40, 4, 2, D)
    hold(K, (k.float().clamp(-2, 2) * k_size).to(BF), v, (q.float() * q_size).to(BF), pos, which="prefill")


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("which", ["prefill", "decode"])
def test_rows_of_queries_of_different_sizes(K, D, which):
    """Each row has a size of its own, an outlying channel a hundred times the others'; one row is zero."""
    k, v, q, pos = inputs(D, 300, 8, 4, 2, D)
    q = q.float()
    q[..., 5] *= 100
    k = k.float()
    k[..., 5] /= 100
    q = q * torch.tensor([1e-12, 1e-3, 1.0, 30.0, 1e-6, 1e-4, 0.0, 1e-30])[:, None, None]
    hold(K, k.to(BF), v, q.to(BF), pos, which=which)


@pytest.mark.parametrize("D", [128, 256])
def test_keys_whose_offsets_cancel(K, D):
    """Half of the tokens have keys of 20000 in one group and -20000 in another, whose products with q cancel."""
    g = torch.Generator().manual_seed(D)
    Hq, Hkv, n = 4, 2, 300
    q = torch.randn(1, Hq, D, generator=g)
    q = (q * 64).round() / 64
    q = torch.cat([q[..., :64], q[..., :64].flip(-1), q[..., 128:]], -1)[..., :D].to(BF)          # equal sums over the first two groups
    k, v = torch.randn(n, Hkv, D, generator=g), rows(g, n, Hkv, D)
    k[::2, :, :64], k[::2, :, 64:128] = 20000.0, -20000.0
    hold(K, k.to(BF), v, q, torch.tensor([n - 1]), which="decode")


# ---- bytes that no row sees -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("free", [0x7F, 0xFF, 0x80])
def test_bytes_in_front_of_the_window(K, D, free):
    """Nothing was ever written there: huge scales (0x7F: 3.4e38), NaN, whatever."""
    n, T, window, Hq, Hkv = 300, 40, 30, 4, 2
    g = torch.Generator().manual_seed(D)
    k, v, q = rows(g, n, Hkv, D), rows(g, n, Hkv, D), torch.randn(T, Hq, D, generator=g).to(BF)
    pos = torch.arange(n - T, n)
    pool = Filled(k, v, free, first=n - T - window + 1)
    want, tol = attention(q, pool.k, pool.v, pos, window, prefill=True)
    for splits in (1, 2):
        assert worst(prefill(K, pool, q, n - T, window, splits=splits), want, tol) <= 1
    want, tol = attention(q, pool.k, pool.v, pos, window)
    assert worst(decode(K, pool, q[:8], pos[:8], window), want[:8], tol[:8]) <= 1
    assert math.isfinite(float(want.abs().max()))
