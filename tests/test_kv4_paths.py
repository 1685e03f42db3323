"""The 4-bit KV cache between ranks, and the bound that its plans keep (CPU)."""
import os
import socket
import sys
from types import SimpleNamespace

import pytest
import torch
import torch.multiprocessing as mp

from r4dx_b200.quant import kv4

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_no_warp_adds_up_more_than_4096_tokens():
    """Tensor-core sums round towards zero at each block; the decode kernel's warps take the blocks of their CTA in turn, the CTAs equal shares."""
    from r4dx_b200.ops import kernels as K
    for D in (64, 128, 256):
        for rows in (1, 6, 8, 24, 48, 192):
            for heads in (1, 4, 8):
                for batch in (1, 2, 16, 64):
                    for length in (1, 9, 64, 512, 600, 4096, 8192, 16384, 65536, 131072):
                        splits, chunk, _ = K.kv4_splits(rows, heads, batch, length, D)
                        tile = K.kv4_row_tile(rows, D, length)
                        warps = K._KV4_CTAS[D, tile][0]
                        for blocks in {length, (length + 1) // 2}:
                            per = -(-blocks // max(1, min(splits, -(-blocks // chunk))))
                            take = 2 if tile == 8 and per > warps else 1            # blocks that a warp takes at a time
                            assert 16 * take * -(-per // (warps * take)) <= 4096, (D, rows, heads, batch, blocks, splits)


def _rows(layer, Hkv, D, n):
    g = torch.Generator().manual_seed(layer)
    return [(torch.randn(n, Hkv, D, generator=g) * s).to(torch.bfloat16) for s in (1.0, 0.3)]


def _reshard(rank, world, port, results):
    sys.path.insert(0, ROOT)
    import datetime
    import torch.distributed as dist
    from r4dx_b200.config import tiny_hybrid_config
    from r4dx_b200.parallel.pp import reshard_to_tp
    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=world, timeout=datetime.timedelta(seconds=60))
    cfg = tiny_hybrid_config()
    part, n, blocks = cfg.shard(world, rank), 37, 5
    owner = {i: int(i >= cfg.num_hidden_layers // 2) for i in range(cfg.num_hidden_layers)}
    attention = [i for i in range(cfg.num_hidden_layers) if cfg.is_attention_layer(i)]
    linear = [i for i in range(cfg.num_hidden_layers) if not cfg.is_attention_layer(i)]

    def model(c, layers):
        return SimpleNamespace(pos=0, pending_rows=1, device=torch.device("cpu"), buf=SimpleNamespace(n_replay=torch.ones(1)),
                               kv={i: torch.full(kv4.pool_shape(blocks, c.num_key_value_heads, c.head_dim), 0xFF, dtype=torch.uint8) for i in layers if i in attention},
                               gdn_state={i: torch.zeros(c.linear_num_value_heads, c.linear_key_head_dim, c.linear_key_head_dim) for i in layers if i in linear},
                               ring={i: torch.zeros(32, c.conv_dim) for i in layers if i in linear})

    stage, tp = model(cfg, [i for i in owner if owner[i] == rank]), model(part, list(owner))
    stage.pos, stage.pending_rows = n, 0
    pos = torch.arange(n)
    for i, pool in stage.kv.items():
        kv4.write_rows(pool, *_rows(i, cfg.num_key_value_heads, cfg.head_dim, n), pos // 16, pos % 16)
    for i in stage.gdn_state:
        stage.gdn_state[i] += torch.arange(cfg.linear_num_value_heads)[:, None, None]
    reshard_to_tp(cfg, stage, tp, world, rank, owner)
    h = part.num_key_value_heads
    first = rank * h if cfg.num_key_value_heads >= world else 0
    ok = tp.pos == n and len(attention) > 0
    for i in attention:
        for got, x in zip(kv4.read_rows(tp.kv[i], pos // 16, pos % 16), _rows(i, cfg.num_key_value_heads, cfg.head_dim, n)):
            ok = ok and torch.equal(got, kv4.round_trip(x[:, first:first + h]))
        ok = ok and bool((tp.kv[i][(n + 15) // 16:] == 0xFF).all())
    results.put((rank, ok))
    dist.barrier()
    dist.destroy_process_group()


def test_pools_handed_over_from_pipeline_stages():
    """After a pipelined prompt every tensor-parallel rank has its heads of every layer's rows, and no other block is touched."""
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    results = ctx.Queue()
    ranks = [ctx.Process(target=_reshard, args=(r, 2, port, results)) for r in range(2)]
    for p in ranks:
        p.start()
    got = dict(results.get(timeout=120) for _ in ranks)
    for p in ranks:
        p.join(60)
    assert got == {0: True, 1: True}


@pytest.mark.parametrize("D", [64, 128, 256])
def test_workload_and_library_write_the_same_values(D):
    """The plain writer of perf/operators.py and that of quant/kv4.py: every row stands for the same values, constant groups among them."""
    sys.path.insert(0, ROOT)
    from perf import operators as P
    g = torch.Generator().manual_seed(D)
    k, v = ((torch.randn(20, 2, D, generator=g)).to(torch.bfloat16) for _ in range(2))
    k[3, 1, :64] = 1.5
    v[7] = 0.0
    block, tok = torch.tensor([2] * 16 + [0] * 4), torch.arange(20) % 16
    a, b = (torch.zeros(kv4.pool_shape(3, 2, D), dtype=torch.uint8) for _ in range(2))
    kv4.write_rows(a, k, v, block, tok)
    P.put(b, 0, D, block, tok, k)
    P.put(b, 1, D, block, tok, v)
    for x, y in zip(kv4.read_rows(a, block, tok), kv4.read_rows(b, block, tok)):
        assert torch.equal(x, y)
    assert torch.equal(kv4.read_rows(a, block, tok)[0], P.get_rows(b, 0, D, block, tok))
