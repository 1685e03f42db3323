"""The 4-bit paged KV cache on the GPU: rows written and read back bit by bit against the format's definition, attention against 64-bit
attention over the values that the cache stands for."""
import math

import pytest
import torch

from r4dx_b200.quant import kv4

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
NAN = float("nan")


@pytest.fixture(scope="module")
def K():
    from r4dx_b200.ops import kernels
    return kernels


def rows(g, n, heads, D, spread=1.0):
    """bf16 rows as caches hold them: some channels louder than others."""
    loud = torch.exp(0.5 * torch.randn(1, heads, D, generator=g))
    return (torch.randn(n, heads, D, generator=g) * loud * spread).to(BF)


class Pool:
    """A pool filled by the plain writer through shuffled block tables; every byte that no row owns is 0xFF (scales and codes of NaN)."""

    def __init__(self, D, Hkv, lengths, seed=0, extra=2, spread=1.0):
        g = torch.Generator().manual_seed(seed)
        need = [(n + 15) // 16 for n in lengths]
        blocks = sum(need) + extra
        order = torch.randperm(blocks, generator=g).to(torch.int32)
        self.tables = torch.full((len(lengths), max(need) + 1), -1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(need):
            self.tables[i, :n] = order[at:at + n]
            at += n
        self.spare = order[at:]
        self.cache = torch.full(kv4.pool_shape(blocks, Hkv, D), 0xFF, dtype=torch.uint8)
        self.k, self.v = [], []
        for i, n in enumerate(lengths):
            k, v = rows(g, n, Hkv, D), rows(g, n, Hkv, D, spread)
            pos = torch.arange(n)
            kv4.write_rows(self.cache, k, v, self.tables[i][pos // 16], pos % 16)
            self.k.append(kv4.round_trip(k).double())
            self.v.append(kv4.round_trip(v).double())


def attention(q, k, v, pos, window=0, limit=None):
    """64-bit rows [T, Hq, D] over keys [n, Hkv, D]; zeros for a row that sees nothing."""
    T, Hq, D = q.shape
    kp = torch.arange(k.shape[0])[None]
    last = pos if limit is None else torch.maximum(pos, limit)
    hidden = (kp > last[:, None]) | ((kp <= pos[:, None] - window) if window else torch.zeros_like(kp > pos[:, None]))
    g = Hq // k.shape[1]
    s = torch.einsum("thd,nhd->htn", q.double(), k.repeat_interleave(g, 1)) / math.sqrt(D)
    p = s.masked_fill(hidden[None], -math.inf).softmax(-1)
    p = torch.where(hidden.all(1)[None, :, None], 0.0, p)
    o = torch.einsum("htn,nhd->thd", p.masked_fill(hidden[None], 0.0), torch.where(hidden.all(0)[:, None, None], 0.0, v).repeat_interleave(g, 1))
    return o


def check(out, want, v, slack=0.0):
    """Outputs are rounded to bf16 (2^-8 of them).  Probabilities times scales are rounded to bf16 or fp16: 2^-8 of the codes' share of
    each value, at most 8 steps.  ``slack``: what rounding the operands of the scores adds.  In the 2-norm the output's rounding is
    0.42 of its bound (uniform error, uniform mantissa: 2^-8 / sqrt(3) * 0.72) and the products' no more than that: 2^-8 covers both."""
    out, want = out.double().cpu(), want.cpu()
    step = float((v.amax() - v.amin()) / 15) if v.numel() else 0.0
    bound = 2.0 ** -8 * want.abs() + 2.0 ** -8 * 8 * step + slack + 1e-6
    assert torch.isfinite(out).all()
    assert ((out - want).abs() <= bound).all(), float(((out - want).abs() - bound).max())
    if want.norm() > 0:
        assert (out - want).norm() <= 2.0 ** -8 * want.norm(), float((out - want).norm() / want.norm())


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("T,Hkv,batch", [(1, 1, False), (5, 3, False), (100, 2, False), (1203, 4, False), (7, 2, True)])
def test_written_rows_are_the_formats_bit_for_bit(K, D, T, Hkv, batch):
    """Every byte of the pool, those of other rows among them; rows with NaN, infinities, equal values, huge and tiny ranges."""
    g = torch.Generator().manual_seed(T + D)
    k, v = rows(g, T, Hkv, D), rows(g, T, Hkv, D, 0.5)
    special = [NAN, math.inf, -math.inf, 3.0e38, -1e5, 1e-38, 0.0, -0.0]
    for i in range(0, T, 3):
        k[i, i % Hkv, (7 * i) % D] = special[i // 3 % len(special)]
    v[0] = 2.5
    v[T // 2, 0] = 0.0
    v[T - 1, Hkv - 1, :64] *= 1e-30
    if batch:
        lengths = [5 + 40 * i for i in range(T)]
        slot = torch.randperm(T, generator=g).to(torch.int32)
        pos = torch.tensor([lengths[s] - 1 for s in slot.tolist()], dtype=torch.int32)
    else:
        lengths, slot = [T + 37], None
        pos = (37 + torch.randperm(T, generator=g)).to(torch.int32)
    pool = Pool(D, Hkv, lengths, seed=T)
    tables = pool.tables if batch else pool.tables[0].contiguous()
    got = pool.cache.cuda()
    K.kv4_write(k.cuda(), v.cuda(), pos.cuda(), tables.cuda(), got, row_slot=slot.cuda() if batch else None)
    entries = tables[slot.long(), pos.long() // 16] if batch else tables[pos.long() // 16]
    kv4.write_rows(pool.cache, k, v, entries, pos % 16)
    want_k, want_v = kv4.read_rows(pool.cache, entries, pos % 16)
    rk, rv = K.kv4_read(got, tables.cuda(), pos.cuda(), row_slot=slot.cuda() if batch else None)
    for a, b in ((rk, want_k), (rv, want_v)):
        assert torch.equal(a.cpu().isnan(), b.isnan())
        assert torch.equal(a.cpu().nan_to_num(), b.to(BF).nan_to_num())
    # bytes: NaN pairs may differ in their bits, codes of NaN groups and the sign of a zero low end too
    finite = ~want_k.isnan().flatten(1).any(1)
    words, ref = got.cpu().view(torch.int32), pool.cache.view(torch.int32)
    diff = (words != ref).nonzero()
    bad_rows = {(int(entries[r]), int(pos[r]) % 16) for r in range(T) if not bool(finite[r])}
    places = {kv4.word_places(D, False)[t, w].item(): t for t in range(16) for w in range(D // 8)}
    for b, h, part, at in diff.tolist():
        token = places[at] if at < 2 * D and part == 0 else ((at - 2 * D) // (D // 64) if at >= 2 * D else None)
        zero_low = at >= 2 * D and (int(words[b, h, part, at]) ^ int(ref[b, h, part, at])) & 0xFFFFFFFF == 0x80000000
        assert (token is not None and (b, token) in bad_rows) or zero_low, (b, h, part, at)


def test_rows_without_a_place_are_not_written_and_read_as_nan(K):
    D, Hkv = 128, 2
    pool = Pool(D, Hkv, [40, 33], seed=3)
    tables = pool.tables.clone()
    tables[1, 0] = 999                                     # beyond the pool
    g = torch.Generator().manual_seed(1)
    pos = torch.tensor([-1, 16 * tables.shape[1], 47, 3, 17, 20, -(1 << 31), (1 << 31) - 1, 8], dtype=torch.int32)
    slot = torch.tensor([0, 0, 0, 1, 2, -1, 0, 0, 0], dtype=torch.int32)         # position 47: in the table's last block of 40 tokens
    k, v = rows(g, 9, Hkv, D), rows(g, 9, Hkv, D)
    got = pool.cache.cuda()
    K.kv4_write(k.cuda(), v.cuda(), pos.cuda(), tables.cuda(), got, row_slot=slot.cuda())
    kv4.write_rows(pool.cache, k[[2, 8]], v[[2, 8]], tables[0][pos[[2, 8]].long() // 16], pos[[2, 8]] % 16)
    assert torch.equal(got.cpu(), pool.cache)
    rk, rv = K.kv4_read(got, tables.cuda(), pos.cuda(), row_slot=slot.cuda())
    there = torch.tensor([False, False, True, False, False, False, False, False, True])
    for x in (rk, rv):
        assert torch.equal(x.cpu().isnan().all(-1).all(-1), ~there) and not x.cpu()[there].isnan().any()


@pytest.mark.parametrize("D,Hq,Hkv,rot,norm,gate,T,start", [(256, 6, 2, 64, True, True, 1, 9), (256, 24, 4, 64, True, True, 130, 77),
                                                        (128, 8, 8, 128, False, False, 3, 100000), (64, 4, 1, 64, True, False, 33, 0),
                                                        (128, 5, 1, 0, True, False, 2, 5), (64, 2, 2, 22, False, True, 1500, 31)])
def test_precore_norms_rotates_and_quantises(K, D, Hq, Hkv, rot, norm, gate, T, start):
    """q against 64 bits, rounded to bf16.  k: a group's step s = range / 15; rounding k to bf16 moves it by 2^-8 of its size, its code by
    half a step, the scale's rounding clips 15 * 2^-8 of a step, and what is read is rounded by 2^-8 again."""
    g = torch.Generator().manual_seed(T)
    theta, total = 1e6, start + T
    qs = 2 * D if gate else D
    qg, k, v = torch.randn(T, Hq, qs, generator=g).to(BF), rows(g, T, Hkv, D), rows(g, T, Hkv, D)
    qn, kn = ((0.1 * torch.randn(D, generator=g)).to(BF) for _ in range(2)) if norm else (None, None)
    first = start // 16
    blocks = (total + 15) // 16 - first
    table = torch.full(((total + 15) // 16 + 2,), -1, dtype=torch.int32)
    table[first:first + blocks] = torch.randperm(blocks, generator=g).to(torch.int32)
    cache = K.kv4_cache(blocks, Hkv, D)
    pos = torch.arange(start, total, dtype=torch.int32)
    q = torch.full((T, Hq, D), NAN, dtype=BF, device="cuda")
    dev = lambda x: None if x is None else x.cuda()  # noqa: E731
    K.attn_precore_kv4(qg.cuda(), k.cuda(), v.cuda(), dev(qn), dev(kn), pos.cuda(), table.cuda(), q, cache, T, Hq, Hkv, D, rot, theta, q_stride=qs)

    def turned(x, w):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * (1 + w.double())
        h = rot // 2
        a = pos.double()[:, None] * theta ** (-2.0 * torch.arange(h, dtype=torch.float64) / max(rot, 1))
        c, s = a.cos()[:, None], a.sin()[:, None]
        return torch.cat([x[..., :h] * c - x[..., h:rot] * s, x[..., h:rot] * c + x[..., :h] * s, x[..., rot:]], -1)

    want = turned(qg[..., :D], qn)
    assert ((q.double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-6).all()
    rk, rv = K.kv4_read(cache, table.cuda(), pos.cuda())
    assert torch.equal(rv.cpu(), kv4.round_trip(v).to(BF))
    want = turned(k, kn)
    step = ((want.unflatten(-1, (-1, 64)).amax(-1) - want.unflatten(-1, (-1, 64)).amin(-1)) / 15).repeat_interleave(64, -1)
    bound = (0.5 + 15 * 2.0 ** -8) * 1.01 * step + 2 * 2.0 ** -8 * (want.abs() + step)
    assert ((rk.double().cpu() - want).abs() <= bound).all()


DECODE = [
    # D, Hq, Hkv, T, ctx, window, gated, splits
    (256, 24, 4, 1, 1, 0, True, None), (256, 24, 4, 1, 16, 0, True, None), (256, 8, 2, 1, 17, 0, True, 1), (256, 16, 2, 1, 1500, 0, True, None),
    (256, 24, 4, 8, 700, 0, True, None), (256, 6, 1, 3, 333, 100, False, 7), (128, 32, 8, 1, 2049, 0, False, None), (128, 5, 5, 2, 130, 0, True, 3),
    (128, 9, 1, 4, 4000, 513, False, None), (64, 32, 8, 1, 129, 0, False, 2), (64, 4, 4, 8, 40, 9, True, None), (64, 64, 1, 32, 260, 0, False, None),
    (128, 32, 8, 1, 12001, 0, True, None), (256, 24, 4, 1, 13000, 3000, False, None), (64, 8, 1, 6, 20000, 0, False, None),
    (128, 3, 3, 1, 900, 1, False, None), (256, 2, 1, 5, 5, 0, False, 1), (256, 2, 2, 1, 9000, 0, True, None),
]


@pytest.mark.parametrize("D,Hq,Hkv,T,ctx,window,gated,splits", DECODE)
def test_decode_attention(K, D, Hq, Hkv, T, ctx, window, gated, splits):
    g = torch.Generator().manual_seed(ctx + T)
    pool = Pool(D, Hkv, [ctx], seed=ctx)
    q = torch.randn(T, Hq, D, generator=g).to(BF)
    qg = torch.randn(T, Hq, 2 * D, generator=g).to(BF)
    pos = torch.arange(ctx - T, ctx, dtype=torch.int32)
    out = torch.full((T, Hq, D), NAN, dtype=BF, device="cuda")
    K.attn_decode_kv4(q.cuda(), qg.cuda() if gated else None, pool.cache.cuda(), pool.tables[0].cuda(), pos.cuda(), out, T, Hq, Hkv, D, gated=gated,
                      window=window, splits=splits)
    K.check_gemm_status(out.device)
    want = attention(q, pool.k[0], pool.v[0], pos.long(), window)
    if gated:
        want = want * torch.sigmoid(qg[..., D:].double())
    check(out, want, pool.v[0])
    again = torch.full_like(out, NAN)
    K.attn_decode_kv4(q.cuda(), qg.cuda() if gated else None, pool.cache.cuda(), pool.tables[0].cuda(), None, again, T, Hq, Hkv, D, gated=gated,
                      window=window, splits=splits, pos0=ctx - T)
    assert torch.equal(out, again)


@pytest.mark.parametrize("D,Hq,Hkv,window,splits", [(256, 24, 4, 0, None), (128, 8, 2, 0, 4), (64, 32, 8, 50, None), (128, 16, 1, 0, 1)])
def test_batched_decode_with_padding_and_missing_pages(K, D, Hq, Hkv, window, splits):
    """Rows of sequences of all lengths; a padding row (position -1) gives zeros; a slot or a page that does not exist gives NaN to the rows
    that see it and to no others (a missing page behind the window or behind the row's position is nobody's)."""
    lengths = [1, 700, 16, 33, 129, 300, 64, 1000]
    pool = Pool(D, Hkv, lengths, seed=5)
    g = torch.Generator().manual_seed(D)
    tables = pool.tables.clone()
    tables[3, 1] = 10 ** 6                                  # position 20 sees it
    tables[4, 8] = -5                                       # position 100 does not
    slot = torch.tensor([7, 0, 3, 1, 9, 4, 2, 6, 5], dtype=torch.int32)
    pos = torch.tensor([999, 0, 20, 350, 5, 100, -1, 63, 299], dtype=torch.int32)
    B = len(slot)
    q, qg = torch.randn(B, Hq, D, generator=g).to(BF), torch.randn(B, Hq, 2 * D, generator=g).to(BF)
    out = torch.full((B, Hq, D), NAN, dtype=BF, device="cuda")
    K.attn_decode_kv4(q.cuda(), qg.cuda(), pool.cache.cuda(), tables.cuda(), pos.cuda(), out, B, Hq, Hkv, D, window=window, row_slot=slot.cuda(),
                      splits=splits)
    K.check_gemm_status(out.device)
    out = out.cpu()
    for b in range(B):
        if int(slot[b]) in (9, 3):
            assert out[b].isnan().all(), b
        elif int(pos[b]) < 0:
            assert (out[b] == 0).all(), b
        else:
            s = int(slot[b])
            want = attention(q[b:b + 1], pool.k[s], pool.v[s], pos[b:b + 1].long(), window) * torch.sigmoid(qg[b:b + 1, :, D:].double())
            check(out[b:b + 1], want, pool.v[s])


def test_decode_window_past_freed_pages_and_before_the_table_ends(K):
    """Pages behind a window may be gone; rows beyond the table see a page that is not there."""
    D, Hq, Hkv, ctx, window = 128, 8, 2, 500, 40
    pool = Pool(D, Hkv, [ctx], seed=9)
    table = pool.tables[0].clone()
    table[:(ctx - 4 - window + 1) // 16] = -1
    g = torch.Generator().manual_seed(2)
    q = torch.randn(4, Hq, D, generator=g).to(BF)
    pos = torch.arange(ctx - 4, ctx, dtype=torch.int32)
    out = torch.empty(4, Hq, D, dtype=BF, device="cuda")
    args = (4, Hq, Hkv, D, False, window)
    K.attn_decode_kv4(q.cuda(), None, pool.cache.cuda(), table.cuda(), pos.cuda(), out, *args)
    check(out, attention(q, pool.k[0], pool.v[0], pos.long(), window), pool.v[0])
    K.attn_prefill_kv4(q.cuda(), None, pool.cache.cuda(), table.cuda(), out, 4, Hq, Hkv, D, ctx - 4, False, window)
    check(out, attention(q, pool.k[0], pool.v[0], pos.long(), window), pool.v[0], slack=score_slack(q, pool.k[0], pool.v[0]))
    short = table[:31].contiguous()                         # positions 496 .. lie in block 31
    K.attn_decode_kv4(q.cuda(), None, pool.cache.cuda(), short.cuda(), pos.cuda(), out, *args)
    assert out.isnan().all()
    K.attn_prefill_kv4(q.cuda(), None, pool.cache.cuda(), short.cuda(), out, 4, Hq, Hkv, D, ctx - 4, False, window)
    assert out.isnan().all()
    K.check_gemm_status(out.device)


def score_slack(q, k, v):
    """Prefill rounds q and the keys to fp16 (2^-11 each): a score moves by at most 2 * 2^-11 of the sum of |q k|, the output by twice that
    of the largest value; probabilities and values are rounded to fp16 too."""
    a = float((q.double().abs().amax(0).amax(0) * k.abs().amax(0).amax(0)).sum()) / math.sqrt(q.shape[-1])
    return float(v.abs().max()) * (2 * 2 * 2.0 ** -11 * a + 2 * 2.0 ** -11 + 1e-4)


PREFILL = [
    # D, Hq, Hkv, T, pos0, window, gated, splits
    (256, 6, 1, 1, 0, 0, True, None), (256, 24, 4, 333, 0, 0, True, None), (256, 3, 1, 129, 127, 0, True, None), (128, 8, 2, 260, 500, 130, False, None),
    (128, 5, 5, 257, 300, 64, True, None), (64, 32, 8, 100, 29, 0, False, None), (64, 3, 3, 300, 1000, 17, True, None), (256, 2, 2, 17, 2000, 0, False, None),
    (64, 4, 2, 513, 0, 0, True, None), (128, 2, 1, 40, 16, 1, False, None), (256, 4, 2, 128, 128, 0, False, None),
    (256, 24, 4, 16, 3000, 0, True, None), (128, 8, 2, 130, 2500, 0, False, 4), (64, 6, 2, 140, 900, 300, True, 5), (256, 2, 1, 300, 200, 0, True, 7),
    # the kernel itself where the decode kernel would take the call
    (256, 24, 4, 1, 0, 0, True, 1), (64, 4, 2, 5, 40, 0, True, 1), (128, 3, 1, 31, 700, 90, True, 2), (256, 5, 1, 32, 127, 0, False, 1), (128, 8, 2, 1, 4000, 0, True, 6),
]


@pytest.mark.parametrize("D,Hq,Hkv,T,pos0,window,gated,splits", PREFILL)
def test_prefill_attention(K, D, Hq, Hkv, T, pos0, window, gated, splits):
    g = torch.Generator().manual_seed(T + pos0)
    pool = Pool(D, Hkv, [pos0 + T], seed=T)
    q, qg = torch.randn(T, Hq, D, generator=g).to(BF), torch.randn(T, Hq, 2 * D, generator=g).to(BF)
    out = torch.full((T, Hq, D), NAN, dtype=BF, device="cuda")
    K.attn_prefill_kv4(q.cuda(), qg.cuda() if gated else None, pool.cache.cuda(), pool.tables[0].cuda(), out, T, Hq, Hkv, D, pos0, gated, window,
                       splits=splits)
    K.check_gemm_status(out.device)
    want = attention(q, pool.k[0], pool.v[0], torch.arange(pos0, pos0 + T), window)
    if gated:
        want = want * torch.sigmoid(qg[..., D:].double())
    check(out, want, pool.v[0], slack=score_slack(q, pool.k[0], pool.v[0]))


@pytest.mark.parametrize("D,window", [(64, 24), (256, 100), (128, 0)])
def test_prefill_key_limits(K, D, window):
    """Rows of an image block see the whole block."""
    Hq, Hkv, T, pos0 = 4, 2, 150, 61
    g = torch.Generator().manual_seed(D)
    pool = Pool(D, Hkv, [pos0 + T], seed=D)
    limit = torch.full((T,), -1, dtype=torch.int32)
    limit[20:90] = pos0 + 89
    q = torch.randn(T, Hq, D, generator=g).to(BF)
    out = torch.empty(T, Hq, D, dtype=BF, device="cuda")
    K.attn_prefill_kv4(q.cuda(), None, pool.cache.cuda(), pool.tables[0].cuda(), out, T, Hq, Hkv, D, pos0, False, window, limit.cuda())
    want = attention(q, pool.k[0], pool.v[0], torch.arange(pos0, pos0 + T), window, limit.long())
    check(out, want, pool.v[0], slack=score_slack(q, pool.k[0], pool.v[0]))


@pytest.mark.parametrize("D", [64, 128, 256])
def test_nan_keys_and_values_reach_the_rows_that_see_them_only(K, D):
    """A key at position 70 (head 0) and a value at position 75 (first 64 channels of head 1) are NaN: rows before them are as if nothing
    were there, rows after are NaN (of the value: in its channels), rows whose window has passed them are clean again."""
    Hq, Hkv, n, window = 4, 2, 200, 30
    g = torch.Generator().manual_seed(D)
    pool = Pool(D, Hkv, [n], seed=D)
    k, v = rows(g, 2, Hkv, D), rows(g, 2, Hkv, D)
    k[0, 0, 3], v[1, 1, 5] = NAN, NAN
    pos = torch.tensor([70, 75])
    kv4.write_rows(pool.cache, k, v, pool.tables[0][pos // 16], pos % 16)
    for i, p in enumerate(pos.tolist()):
        pool.k[0][p], pool.v[0][p] = kv4.round_trip(k[i]).double().nan_to_num(), kv4.round_trip(v[i]).double().nan_to_num()
    q = torch.randn(n, Hq, D, generator=g).to(BF)
    at = torch.arange(n)
    want = attention(q, pool.k[0], pool.v[0], at, window)
    nan = torch.zeros(n, Hq, D, dtype=torch.bool)
    nan[70:70 + window, :2] = True
    nan[75:75 + window, 2:, :64] = True
    cache, table = pool.cache.cuda(), pool.tables[0].cuda()
    out = torch.empty(n, Hq, D, dtype=BF, device="cuda")
    for splits in (1, 2):
        K.attn_prefill_kv4(q.cuda(), None, cache, table, out, n, Hq, Hkv, D, 0, False, window, splits=splits)
        assert torch.equal(out.cpu().isnan(), nan), splits
        check(out.cpu().masked_fill(nan, 0.0), want.masked_fill(nan, 0.0), pool.v[0], slack=score_slack(q, pool.k[0], pool.v[0]))
    for first in (64, 68, 72, 96, 104):
        r = slice(first, first + 8)
        K.attn_decode_kv4(q[r].contiguous().cuda(), None, cache, table, at[r].int().cuda(), out[:8], 8, Hq, Hkv, D, False, window)
        assert torch.equal(out[:8].cpu().isnan(), nan[r]), first
        check(out[:8].cpu().masked_fill(nan[r], 0.0), want[r].masked_fill(nan[r], 0.0), pool.v[0])
    K.check_gemm_status(out.device)


def test_rows_in_any_order_of_positions(K):
    """Rows of one sequence need not be sorted, some may be padding, some beyond the table; sixteen of them take two row tiles."""
    D, Hq, Hkv, n = 128, 4, 2, 300
    g = torch.Generator().manual_seed(12)
    pool = Pool(D, Hkv, [n], seed=12)
    pos = torch.tensor([299, 0, -1, 17, 17, 150, 16, 5, -7, 299, 31, 32, 128, 1, 2, 3], dtype=torch.int32)
    q = torch.randn(16, Hq, D, generator=g).to(BF)
    out = torch.full((16, Hq, D), NAN, dtype=BF, device="cuda")
    for window in (0, 20):
        K.attn_decode_kv4(q.cuda(), None, pool.cache.cuda(), pool.tables[0].cuda(), pos.cuda(), out, 16, Hq, Hkv, D, False, window)
        check(out, attention(q, pool.k[0], pool.v[0], pos.long(), window), pool.v[0])
        assert (out[2] == 0).all() and (out[8] == 0).all()
    far = pos.clone()
    far[5] = 2 ** 31 - 1
    K.attn_decode_kv4(q.cuda(), None, pool.cache.cuda(), pool.tables[0].cuda(), far.cuda(), out, 16, Hq, Hkv, D, False, 20)
    assert torch.equal(out.isnan().flatten(1).all(1).cpu(), far == 2 ** 31 - 1)
    K.check_gemm_status(out.device)


@pytest.mark.parametrize("D,splits", [(64, None), (128, 3), (256, None), (256, 1)])
def test_positions_far_behind_the_table(K, D, splits):
    """Rows whose position no table has are NaN and cost no more than a full table; the others are what they are without them."""
    Hq, Hkv, n = 4, 2, 300
    g = torch.Generator().manual_seed(13)
    pool = Pool(D, Hkv, [n], seed=13)
    end = 16 * pool.tables.shape[1]
    pos = torch.tensor([299, end, 2 ** 31 - 1, -1, 40, 2 ** 30], dtype=torch.int32)
    q = torch.randn(6, Hq, D, generator=g).to(BF)
    for window in (0, 33):
        out = torch.zeros(6, Hq, D, dtype=BF, device="cuda")
        args = (q.cuda(), None, pool.cache.cuda(), pool.tables[0].cuda(), pos.cuda(), out, 6, Hq, Hkv, D, False, window)
        ms = []
        for _ in range(5):
            start, stop = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            K.attn_decode_kv4(*args, splits=splits)
            stop.record()
            stop.synchronize()
            ms.append(start.elapsed_time(stop))
        K.check_gemm_status(out.device)
        assert min(ms) < 5.0                                # (2^27 missing blocks, one after the other, are tens of ms and more)
        assert out[[1, 2, 5]].isnan().all() and (out[3] == 0).all()
        want = attention(q[[0, 4]], pool.k[0], pool.v[0], pos[[0, 4]].long(), window)
        check(out[[0, 4]], want, pool.v[0])
        one = torch.zeros(1, Hq, D, dtype=BF, device="cuda")
        K.attn_decode_kv4(q[:1].cuda(), None, pool.cache.cuda(), pool.tables[0].cuda(), None, one, 1, Hq, Hkv, D, False, window, splits=splits,
                          pos0=(1 << 30) - 1)
        assert one.isnan().all()


def test_blocks_beyond_four_gigabytes(K):
    """A pool of 4.7 GB of which only the blocks at its ends are used."""
    D, Hq, Hkv, n = 256, 16, 8, 70
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB of device memory")
    blocks = 130000
    cache = torch.empty(kv4.pool_shape(blocks, Hkv, D), dtype=torch.uint8, device="cuda")
    assert cache.numel() > 1 << 32
    table = torch.tensor([blocks - 1, 0, blocks - 2, 1, blocks - 3], dtype=torch.int32)
    g = torch.Generator().manual_seed(0)
    k, v, q = rows(g, n, Hkv, D), rows(g, n, Hkv, D), torch.randn(n, Hq, D, generator=g).to(BF)
    pos = torch.arange(n, dtype=torch.int32)
    K.kv4_write(k.cuda(), v.cuda(), pos.cuda(), table.cuda(), cache)
    rk, rv = K.kv4_read(cache, table.cuda(), pos.cuda())
    kr, vr = kv4.round_trip(k), kv4.round_trip(v)
    assert torch.equal(rk.cpu(), kr.to(BF)) and torch.equal(rv.cpu(), vr.to(BF))
    want = attention(q, kr.double(), vr.double(), pos.long())
    out = torch.empty(n, Hq, D, dtype=BF, device="cuda")
    K.attn_prefill_kv4(q.cuda(), None, cache, table.cuda(), out, n, Hq, Hkv, D, 0, False)
    check(out, want, vr, slack=score_slack(q, kr.double(), vr.double()))
    K.attn_decode_kv4(q[-5:].contiguous().cuda(), None, cache, table.cuda(), pos[-5:].contiguous().cuda(), out, 5, Hq, Hkv, D, False)
    check(out[:5], want[-5:], vr)


def test_two_streams_at_once_and_rows_behind_the_last_one(K):
    """Calls on two streams with scratch of their own; what lies behind the last row of an output stays as it was."""
    D, Hq, Hkv, n = 256, 24, 4, 3000
    g = torch.Generator().manual_seed(21)
    pools = [Pool(D, Hkv, [n], seed=s) for s in (1, 2)]
    q = torch.randn(2, 1, Hq, D, generator=g).to(BF)
    pos = torch.tensor([n - 1], dtype=torch.int32).cuda()
    state = [(q[i].cuda(), p.cache.cuda(), p.tables[0].cuda(), torch.full((3, Hq, D), 7.0, dtype=BF, device="cuda")) for i, p in enumerate(pools)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for st, (a, c, t, o) in zip(streams, state):
            with torch.cuda.stream(st):
                K.attn_decode_kv4(a, None, c, t, pos, o, 1, Hq, Hkv, D, False)
    torch.cuda.synchronize()
    for i, p in enumerate(pools):
        check(state[i][3][:1], attention(q[i], p.k[0], p.v[0], torch.tensor([n - 1])), p.v[0])
        assert (state[i][3][1:] == 7.0).all()


@pytest.mark.parametrize("D,Hq,Hkv,T,start,splits", [(256, 24, 4, 130, 0, None), (128, 8, 2, 64, 1500, 3), (64, 8, 8, 300, 37, 1)])
def test_calls_in_a_row_see_what_the_calls_before_them_wrote(K, D, Hq, Hkv, T, start, splits):
    """Writer, prompt and read-back one after the other on two streams, rows anew each time: the same bits as with a synchronisation after
    every call (a kernel may start before the one in front of it has ended, but not read its rows)."""
    g = torch.Generator().manual_seed(D + T)
    n, rounds = start + T, 6
    blocks = (n + 15) // 16
    q, k, v = (torch.randn(rounds, rows_, h, D, generator=g).to(BF).cuda() for rows_, h in ((T, Hq), (n, Hkv), (n, Hkv)))
    qg = torch.randn(rounds, T, Hq, 2 * D, generator=g).to(BF).cuda()
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    table = torch.arange(blocks, dtype=torch.int32, device="cuda").flip(0).contiguous()

    def run(cache, after):
        got = []
        for i in range(rounds):
            K.kv4_write(k[i], v[i], pos, table, cache)
            after()
            out = torch.empty(T, Hq, D, dtype=BF, device="cuda")
            K.attn_prefill_kv4(q[i], qg[i], cache, table, out, T, Hq, Hkv, D, start, True, splits=splits)
            after()
            got += [out, *K.kv4_read(cache, table, pos)]
            after()
        return got

    want = run(K.kv4_cache(blocks, Hkv, D), torch.cuda.synchronize)
    streams, caches = [torch.cuda.Stream() for _ in range(2)], [K.kv4_cache(blocks, Hkv, D) for _ in range(2)]
    torch.cuda.synchronize()
    results = []
    for stream, cache in zip(streams, caches):
        with torch.cuda.stream(stream):
            results.append(run(cache, lambda: None))
    torch.cuda.synchronize()
    K.check_gemm_status(want[0].device)
    for got in results:
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    check(want[0].cpu(), attention(q[0].cpu(), kv4.round_trip(k[0].cpu()).double(), kv4.round_trip(v[0].cpu()).double(), torch.arange(start, n))
          * torch.sigmoid(qg[0, ..., D:].cpu().double()), kv4.round_trip(v[0].cpu()).double(),
          slack=score_slack(q[0].cpu(), kv4.round_trip(k[0].cpu()).double(), kv4.round_trip(v[0].cpu()).double()))


@pytest.fixture
def wide_tiles(K, monkeypatch):
    """Every decode call takes the kernel of many rows to a CTA, as calls of many rows over long tables do."""
    monkeypatch.setattr(K, "kv4_row_tile", lambda rows, D, length: 16 if D == 256 else 32)
    K.kv4_splits.cache_clear()
    yield
    K.kv4_splits.cache_clear()


@pytest.mark.parametrize("case", [c for c in DECODE if c[3] > 1 or c[1] // c[2] > 4] + [
    (256, 24, 4, 8, 9000, 0, True, None), (128, 32, 8, 16, 7000, 0, False, None), (64, 12, 2, 32, 3000, 1000, True, None)])
def test_decode_attention_in_wide_row_tiles(K, wide_tiles, case):
    test_decode_attention(K, *case)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_nan_and_missing_blocks_in_wide_row_tiles(K, wide_tiles, D):
    test_nan_keys_and_values_reach_the_rows_that_see_them_only(K, D)
    test_positions_far_behind_the_table(K, D, None)
    test_rows_in_any_order_of_positions(K)


def test_large_scores_and_uniform_attention(K):
    """One key that takes all the weight, late, so that everything before it is scaled away; and equal keys over a long context, where the
    result is a small mean of large terms."""
    D, Hq, Hkv, n = 128, 8, 1, 5000
    pool = Pool(D, Hkv, [n], seed=1)
    q = torch.ones(1, Hq, D, dtype=BF) * 8
    k, v = torch.ones(1, Hkv, D, dtype=BF) * 4, torch.full((1, Hkv, D), 1.5, dtype=BF)
    pos = torch.tensor([n - 2])
    kv4.write_rows(pool.cache, k, v, pool.tables[0][pos // 16], pos % 16)
    pool.k[0][n - 2], pool.v[0][n - 2] = kv4.round_trip(k[0]).double(), kv4.round_trip(v[0]).double()
    out = torch.empty(1, Hq, D, dtype=BF, device="cuda")
    at = torch.tensor([n - 1], dtype=torch.int32)
    K.attn_decode_kv4(q.cuda(), None, pool.cache.cuda(), pool.tables[0].cuda(), at.cuda(), out, 1, Hq, Hkv, D, False)
    check(out, attention(q, pool.k[0], pool.v[0], at.long()), pool.v[0])
    q.zero_()
    K.attn_decode_kv4(q.cuda(), None, pool.cache.cuda(), pool.tables[0].cuda(), at.cuda(), out, 1, Hq, Hkv, D, False)
    check(out, attention(q, pool.k[0], pool.v[0], at.long()), pool.v[0])


def test_captured_calls_follow_the_positions_and_streams(K):
    """write -> decode captured once and replayed as the context grows, on a stream of its own; then the rows read back."""
    D, Hq, Hkv, first, steps = 128, 8, 2, 125, 20
    g = torch.Generator().manual_seed(4)
    pool = Pool(D, Hkv, [first + steps], seed=6)
    k, v, q = rows(g, steps, Hkv, D), rows(g, steps, Hkv, D), torch.randn(steps, Hq, D, generator=g).to(BF)
    blank = pool.cache.clone()
    at = torch.arange(first, first + steps)
    kv4.write_rows(blank, torch.zeros(steps, Hkv, D, dtype=BF), torch.zeros(steps, Hkv, D, dtype=BF), pool.tables[0][at // 16], at % 16)
    cache, table = blank.cuda(), pool.tables[0].cuda()
    sk, sv, sq, sp = (torch.zeros_like(x[:1]).cuda() for x in (k, v, q, torch.zeros(1, dtype=torch.int32)))
    sp.fill_(first)
    out = torch.empty(1, Hq, D, dtype=BF, device="cuda")

    def call():
        K.kv4_write(sk, sv, sp, table, cache)
        K.attn_decode_kv4(sq, None, cache, table, sp, out, 1, Hq, Hkv, D, False)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            call()
        got = []
        for i in range(steps):
            for dst, src in ((sk, k[i:i + 1]), (sv, v[i:i + 1]), (sq, q[i:i + 1]), (sp, torch.tensor([first + i], dtype=torch.int32))):
                dst.copy_(src)
            graph.replay()
            got.append(out.clone())
        rk, rv = K.kv4_read(cache, table, at.int().cuda())
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(rk.cpu(), kv4.round_trip(k).to(BF)) and torch.equal(rv.cpu(), kv4.round_trip(v).to(BF))
    keys, values = pool.k[0].clone(), pool.v[0].clone()
    keys[first:], values[first:] = kv4.round_trip(k).double(), kv4.round_trip(v).double()
    check(torch.cat(got), attention(q, keys, values, at), values)


def test_a_layers_calls_together(K):
    """A prompt's rows enter the cache and attend; then tokens one by one; the prompt's last row by the decode kernel is that of the
    prefill kernel up to their roundings."""
    D, Hq, Hkv, T, rot, theta = 256, 8, 2, 140, 64, 1e7
    g = torch.Generator().manual_seed(8)
    qg, k, v = torch.randn(T + 3, Hq, 2 * D, generator=g).to(BF).cuda(), rows(g, T + 3, Hkv, D).cuda(), rows(g, T + 3, Hkv, D).cuda()
    qn, kn = ((0.1 * torch.randn(D, generator=g)).to(BF).cuda() for _ in range(2))
    cache, table = K.kv4_cache(12, Hkv, D), torch.randperm(12, generator=g).to(torch.int32).cuda()
    pos = torch.arange(T + 3, dtype=torch.int32, device="cuda")
    q, out = torch.empty(T + 3, Hq, D, dtype=BF, device="cuda"), torch.empty(T + 3, Hq, D, dtype=BF, device="cuda")
    K.attn_precore_kv4(qg[:T], k[:T], v[:T], qn, kn, pos[:T], table, q, cache, T, Hq, Hkv, D, rot, theta)
    K.attn_prefill_kv4(q, qg, cache, table, out, T, Hq, Hkv, D, 0)
    one = torch.empty(1, Hq, D, dtype=BF, device="cuda")
    K.attn_decode_kv4(q[T - 1], qg[T - 1], cache, table, pos[T - 1:], one, 1, Hq, Hkv, D)
    for t in range(T, T + 3):
        K.attn_precore_kv4(qg[t], k[t], v[t], qn, kn, pos[t:], table, q[t], cache, 1, Hq, Hkv, D, rot, theta)
        K.attn_decode_kv4(q[t], qg[t], cache, table, pos[t:], out[t], 1, Hq, Hkv, D)
    rk, rv = K.kv4_read(cache, table, pos)
    K.check_gemm_status(out.device)
    tab = table.cpu().long()
    ck, cv = kv4.read_rows(cache.cpu(), tab[pos.cpu().long() // 16], pos.cpu() % 16)
    assert torch.equal(rk.cpu(), ck.to(BF)) and torch.equal(rv.cpu(), cv.to(BF))
    want = attention(q.cpu(), ck.double(), cv.double(), pos.cpu().long()) * torch.sigmoid(qg[..., D:].cpu().double())
    check(out, want, cv, slack=score_slack(q.cpu(), ck.double(), cv.double()))
    check(one, want[T - 1:T], cv)


def test_refusals(K):
    D, Hq, Hkv = 128, 4, 2
    cache = K.kv4_cache(4, Hkv, D)
    table = torch.arange(4, dtype=torch.int32, device="cuda")
    e = lambda *s, dtype=BF: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    pos = e(1, dtype=torch.int32)
    q, qg, k, out = e(1, Hq, D), e(1, Hq, 2 * D), e(1, Hkv, D), e(1, Hq, D)

    def decode(**kw):
        a = dict(q=q, qg=qg, cache=cache, block_table=table, positions=pos, out=out, T=1, Hq=Hq, Hkv=Hkv, D=D)
        K.attn_decode_kv4(**{**a, **kw})

    def prefill(**kw):
        a = dict(q=q, qg=qg, cache=cache, block_table=table, out=out, T=1, Hq=Hq, Hkv=Hkv, D=D, pos0=0)
        K.attn_prefill_kv4(**{**a, **kw})

    def precore(**kw):
        a = dict(qg=qg, k=k, v=k, q_norm=None, k_norm=None, positions=pos, block_table=table, q_out=out, cache=cache, T=1, Hq=Hq, Hkv=Hkv, D=D,
                 rotary_dim=64, theta=1e4)
        K.attn_precore_kv4(**{**a, **kw})

    decode(); prefill(); precore()
    odd = e(1 * Hq * D + 4)[1:1 + Hq * D].view(1, Hq, D)
    bad = [(decode, dict(D=64)), (decode, dict(Hkv=1)), (decode, dict(Hq=3)), (decode, dict(T=2)), (decode, dict(T=0)), (decode, dict(window=-1)),
           (decode, dict(q=q.half())), (decode, dict(q=odd)), (decode, dict(q=q.cpu())), (decode, dict(cache=cache[:, :, :1])),
           (decode, dict(cache=cache.float())), (decode, dict(block_table=table.long())), (decode, dict(block_table=table[None])),
           (decode, dict(positions=pos.long())), (decode, dict(positions=None, pos0=-1)),
           (decode, dict(positions=None, row_slot=pos, block_table=table[None])), (decode, dict(row_slot=pos)), (decode, dict(qg=q)), (decode, dict(qg=None)), (decode, dict(out=out[:, :2])),
           (decode, dict(splits=3, scratch=e(8, dtype=torch.float32))), (decode, dict(splits=0)), (decode, dict(splits=1000)),
           (prefill, dict(D=64)), (prefill, dict(T=2)), (prefill, dict(pos0=-1)), (prefill, dict(q=odd)), (prefill, dict(window=-2)),
           (prefill, dict(pos0=65)), (prefill, dict(pos0=1 << 29)),
           (prefill, dict(key_limit=pos.long())), (prefill, dict(cache=cache.transpose(0, 1))), (prefill, dict(T=0)), (prefill, dict(splits=0)), (prefill, dict(splits=65)),
           (precore, dict(rotary_dim=3)), (precore, dict(rotary_dim=130)), (precore, dict(q_stride=100)), (precore, dict(k=odd[:, :2])), (precore, dict(T=2)),
           (precore, dict(q_norm=e(64))), (precore, dict(Hq=0))]
    for f, kw in bad:
        with pytest.raises((K.KernelError, AttributeError)):
            f(**kw)
    with pytest.raises(K.KernelError):
        K.kv4_write(k, e(1, Hkv, 64), pos, table, cache)
    with pytest.raises(K.KernelError):
        K.kv4_read(cache, table, pos, k=e(1, Hkv, 64))
    with pytest.raises(ValueError):
        K.kv4_cache(4, Hkv, 96)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    assert [x.shape[0] for x in K.kv4_read(cache, table, none)] == [0, 0]
    K.kv4_write(e(0, Hkv, D), e(0, Hkv, D), none, table, cache)
    torch.cuda.synchronize()
