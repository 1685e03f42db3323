"""The 4-bit KV cache's format and the calls that are refused before anything runs (CPU)."""
import math

import pytest
import torch

from r4dx_b200.quant import kv4

BF = torch.bfloat16


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("values", [False, True])
def test_every_word_has_a_place_of_its_own(D, values):
    assert sorted(kv4.word_places(D, values).flatten().tolist()) == list(range(2 * D))


@pytest.mark.parametrize("D", [64, 128, 256])
def test_rows_read_back_as_the_round_trip_and_touch_nothing_else(D):
    g = torch.Generator().manual_seed(D)
    pool = torch.randint(0, 256, kv4.pool_shape(3, 2, D), generator=g, dtype=torch.uint8)
    k, v = torch.randn(20, 2, D, generator=g).to(BF), torch.randn(20, 2, D, generator=g).to(BF)
    block, tok = torch.tensor([2] * 16 + [0] * 4), torch.arange(20) % 16
    before = pool.clone()
    kv4.write_rows(pool, k, v, block, tok)
    rk, rv = kv4.read_rows(pool, block, tok)
    assert torch.equal(rk, kv4.round_trip(k)) and torch.equal(rv, kv4.round_trip(v))
    assert torch.equal(pool[1], before[1])
    free = torch.arange(4, 16)
    for a, b in zip(kv4.read_rows(pool, torch.zeros(12), free), kv4.read_rows(before, torch.zeros(12), free)):
        assert torch.equal(a.nan_to_num(), b.nan_to_num())
    assert torch.equal(kv4.read_rows(torch.zeros_like(pool), block, tok)[0], torch.zeros(20, 2, D))


def test_rounding_is_half_a_step():
    """Half a step, and 15 steps' worth of the scale's rounding (2^-8) at the top code."""
    x = (torch.randn(500, 256, generator=torch.Generator().manual_seed(0)) * 3).to(BF)
    n, s, lo = kv4.quantise(x)
    assert int(n.min()) == 0 and int(n.max()) == 15
    bound = (0.5 + 15 * 2.0 ** -8) * s.float().repeat_interleave(64, -1) * (1 + 2.0 ** -8)
    assert ((kv4.round_trip(x) - x.float()).abs() <= bound).all()


def test_values_at_the_edges():
    x = torch.zeros(6, 64, dtype=BF)
    x[0] = 2.5                                   # one value: exact
    x[1, 3], x[1, 9] = math.inf, -math.inf       # saturate
    x[2, 7] = math.nan
    x[3, 0] = 3e38
    x[4] = torch.linspace(-1e-30, 1e-30, 64).to(BF)
    y = kv4.round_trip(x)
    assert (y[0] == 2.5).all() and (y[5] == 0).all()
    assert y[1, 9] == -32768 and 32768 <= y[1, 3] < 65504 and y[1].isfinite().all()
    assert y[2].isnan().all()
    assert abs(float(y[3, 0]) - 32768) <= 15 * 2.0 ** -8 * 32768 / 15
    assert ((y[4] - x[4].float()).abs() <= 0.6 * 2e-30 / 15).all()


def test_head_dimensions():
    for D in (32, 96, 512):
        with pytest.raises(ValueError):
            kv4.pool_shape(1, 1, D)
    assert kv4.pool_shape(7, 2, 128) == (7, 2, 2, 1152)


def test_calls_without_a_gpu_pool_are_refused():
    from r4dx_b200.ops import kernels as K
    cache = torch.zeros(kv4.pool_shape(2, 1, 64), dtype=torch.uint8)
    table, pos = torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    q = torch.zeros(1, 1, 64, dtype=BF)
    for call in (lambda: K.attn_decode_kv4(q, None, cache, table, pos, q, 1, 1, 1, 64, False), lambda: K.kv4_read(cache, table, pos),
                 lambda: K.kv4_write(q, q, pos, table, cache), lambda: K.attn_prefill_kv4(q, None, cache, table, q, 1, 1, 1, 64, 0, False),
                 lambda: K.attn_precore_kv4(q, q, q, None, None, pos, table, q, cache, 1, 1, 1, 64, 0, 1e4, q_stride=64)):
        with pytest.raises(K.KernelError):
            call()


def test_splits_fill_the_chip_once_and_clusters_fit_it():
    from r4dx_b200.ops import kernels as K
    for rows in (1, 6, 48):
        for heads in (1, 2, 8):
            for batch in (1, 3, 64):
                for length in (1, 8, 9, 600, 5000):
                    for D, most in ((64, 32), (128, 32), (256, 16)):
                        s, chunk, cluster = K.kv4_splits(rows, heads, batch, length, D)
                        least = -(-length // (256 * 16))    # 4096 tokens a warp, 16 warps at most
                        groups = heads * batch * -(-rows // most)
                        assert least <= s <= max(1, 2 * least, min(296, (length + 7) // 8)) and chunk >= 8
                        if batch == 1:
                            assert s <= 2 * least or s * groups <= 296
                        else:
                            assert s <= 2 * least or s * groups <= 592
                        assert not cluster or (1 < s <= 16 and groups <= {16: 7, 9: 15}.get(s, 74))


def test_row_tile_follows_rows_and_table():
    """Few rows and short tables: narrow (8 rows to a CTA); wide where the narrow ones would unpack each block more often than that pays."""
    from r4dx_b200.ops import kernels as K
    for D, wide in ((64, 32), (128, 32), (256, 16)):
        assert {K.kv4_row_tile(r, D, n) for r in (1, 8, 24, 40) for n in (1, 100, 100000)} == {8}
        assert {K.kv4_row_tile(r, D, 64) for r in (32, 128, 384)} == {8}
        assert {K.kv4_row_tile(r, D, 4000) for r in (32, 64, 96, 192, 1000)} == {wide}


def test_flag_of_the_commands():
    from r4dx_b200.cli.args import cli_parser, server_parser
    for parser in (cli_parser(), server_parser()):
        assert parser.parse_args(["--model", "m"]).kv_cache == "fp8"
        assert parser.parse_args(["--model", "m", "--kv-cache", "int4"]).kv_cache == "int4"
        with pytest.raises(SystemExit):
            parser.parse_args(["--model", "m", "--kv-cache", "int3"])


def test_four_stream_family_keeps_its_fp8_cache():
    from types import SimpleNamespace
    from r4dx_b200.cli.loader import _load_qwen4_exp
    with pytest.raises(SystemExit, match="--kv-cache int4"):
        _load_qwen4_exp(SimpleNamespace(tp=1, kv_cache="int4"), None, {}, "m", "m", "cpu")


def test_prefill_shares_fill_the_chip():
    from r4dx_b200.ops import kernels as K
    for D in (64, 128, 256):
        for Hq, Hkv in ((24, 4), (32, 8), (3, 1), (16, 8)):
            for T in (1, 9, 32, 33, 128, 333, 1024, 8192):
                for pos0 in (0, 100, 4000, 29000, 250000):
                    for window in (0, 64, 1024):
                        s = K.kv4_prefill_splits(T, Hq, Hkv, D, pos0, window)
                        keys = min(window + T, pos0 + T) if window else pos0 + T
                        assert 0 <= s <= 64 and (s > 0 or T <= K.KV4_MAX_ROWS) and (s < 2 or s * 256 <= keys + 256 and s * T * Hq * D <= 1 << 26)
    assert K.kv4_prefill_splits(8192, 24, 4, 256, 0, 0) == 1 and K.kv4_prefill_splits(128, 24, 4, 256, 29000, 0) >= 4


def test_entry_points_refuse_bad_arguments_without_a_gpu():
    """Each C entry answers before it touches a pointer or the device."""
    from r4dx_b200 import native
    from r4dx_b200.ops import kernels  # noqa: F401  (signatures)
    L, bad, large = native.cuda(), 10001, 10003
    p, odd = 1 << 20, (1 << 20) + 4

    def decode(q=p, qg=p, cache=p, tables=p, slots_of=None, slots=1, length=4, pool=4, pos=p, pos0=0, scratch=p, out=p, T=1, batch=1, Hq=4, Hkv=2, D=128,
               tile=8, splits=2, chunk=8, cluster=0, window=0):
        return L.r4dxb_attn_decode_kv4(q, qg, cache, tables, slots_of, slots, length, pool, pos, pos0, scratch, out, T, batch, Hq, Hkv, D, tile,
                                       splits, chunk, cluster, window, None, None)

    for kw in (dict(T=0), dict(T=33), dict(batch=2), dict(batch=0), dict(slots_of=p, T=2), dict(Hq=3), dict(Hkv=0), dict(D=96), dict(splits=0),
               dict(splits=257), dict(splits=17, cluster=1), dict(chunk=0), dict(window=-1), dict(length=0), dict(pool=0), dict(slots=0), dict(q=None),
               dict(cache=None), dict(tables=None), dict(pos=None, pos0=-1), dict(pos=None, slots_of=p), dict(out=None), dict(scratch=None), dict(q=odd), dict(cache=odd), dict(out=odd),
               dict(scratch=odd), dict(slots_of=p, batch=70000), dict(tile=16), dict(tile=0), dict(D=256, tile=32), dict(D=64, tile=16)):
        assert decode(**kw) == bad, kw
    assert decode(Hq=1 << 20, Hkv=1 << 16) == large

    def prefill(q=p, qg=p, cache=p, table=p, length=4, pool=4, out=p, T=1, Hq=4, Hkv=2, D=128, pos0=0, window=0, splits=1, scratch=None):
        return L.r4dxb_attn_prefill_kv4(q, qg, cache, table, length, pool, out, T, Hq, Hkv, D, pos0, window, None, splits, scratch, None, None)

    for kw in (dict(T=0), dict(Hq=3), dict(Hq=0), dict(D=32), dict(pos0=-1), dict(pos0=65), dict(pos0=2 ** 31 - 2), dict(window=-1), dict(splits=0), dict(splits=65),
               dict(splits=2), dict(splits=2, scratch=odd), dict(q=odd), dict(qg=odd), dict(out=odd), dict(q=None), dict(cache=None), dict(table=None),
               dict(out=None), dict(length=0), dict(pool=0)):
        assert prefill(**kw) == bad, kw
    assert prefill(Hq=40000, Hkv=1) == large

    def precore(qg=p, k=p, v=p, pos=p, tables=p, slots=1, length=4, pool=4, q=p, cache=p, T=1, Hq=4, Hkv=2, D=128, rot=64, theta=1e4, stride=256):
        return L.r4dxb_attn_precore_kv4(qg, k, v, None, None, pos, tables, None, slots, length, pool, q, cache, T, Hq, Hkv, D, rot, theta, 1e-6, stride, None)

    for kw in (dict(T=0), dict(Hq=-1), dict(Hkv=0), dict(D=80), dict(rot=-2), dict(rot=63), dict(rot=130), dict(theta=0.0), dict(theta=math.nan),
               dict(stride=64), dict(stride=130), dict(qg=None), dict(q=None), dict(k=None), dict(v=None), dict(pos=None), dict(tables=None),
               dict(cache=None), dict(k=odd), dict(cache=odd), dict(q=odd), dict(length=0), dict(pool=0), dict(slots=0)):
        assert precore(**kw) == bad, kw

    def read(cache=p, tables=p, slots=1, length=4, pool=4, pos=p, k=p, v=p, T=1, Hkv=2, D=128):
        return L.r4dxb_kv4_read(cache, tables, None, slots, length, pool, pos, k, v, T, Hkv, D, None)

    for kw in (dict(T=0), dict(Hkv=0), dict(D=48), dict(cache=None), dict(tables=None), dict(pos=None), dict(k=None), dict(v=None), dict(k=odd),
               dict(cache=odd), dict(length=0), dict(pool=0), dict(slots=0)):
        assert read(**kw) == bad, kw
    assert read(Hkv=40000) == large
