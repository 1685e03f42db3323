"""The 4-bit KV cache where the framework itself calls it: the loader and its flag, the drafter head, windows beside single steps, batches of the
writer with norms and rotation (needs a B200)."""
from types import SimpleNamespace

import pytest
import torch

from r4dx_b200.config import tiny_hybrid_config
from r4dx_b200.quant import kv4

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _weights(**kw):
    from r4dx_b200.models.oracle import OracleModel, init_weights
    from r4dx_b200.quant.weights import dequantize_weight_set, quantize_weight_set
    cfg = tiny_hybrid_config()
    q = quantize_weight_set(cfg, init_weights(cfg, 0, **kw))
    dq = dequantize_weight_set(q)
    return cfg, {k: (v.to("cuda") if hasattr(v, "to") else v) for k, v in q.items()}, [OracleModel(cfg, dq, int4_kv=True, act_dtype=t) for t in (None, BF)]


def test_flag_reaches_the_model_through_the_loader():
    from r4dx_b200.cli.loader import load_text_model
    from r4dx_b200.models.hybrid import HybridModel
    from r4dx_b200.quant.weights import synthetic_weight_set
    base = dict(model="synthetic:tiny", layers=0, tp=1, pp=1, hybrid=False, ep=1, max_ctx=256, mtp=0, ngram=0, dflash=None, tokenizer_dir=None,
                prefill_chunk=0, vision="off")
    prompt = torch.randint(0, 200, (45,), generator=torch.Generator().manual_seed(3)).tolist()
    cfg = tiny_hybrid_config()
    for name, per_token in (("int4", 9), ("fp8", 16)):
        tm, _, _ = load_text_model(SimpleNamespace(kv_cache=name, **base), device="cuda:0")
        assert tm.m.kv_cache == name
        assert {t.numel() for t in tm.m.kv.values()} == {(256 // 16 + 1) * cfg.num_key_value_heads * 2 * per_token * cfg.head_dim}
        direct = HybridModel(cfg, synthetic_weight_set(cfg, device="cuda:0", seed=0), max_ctx=256, kv_cache=name)
        got, want = [tm.prefill(prompt)], [direct.prefill(torch.tensor(prompt, dtype=torch.int32))]
        for _ in range(6):
            got.append(tm.decode_step_greedy(got[-1]))
            want.append(direct.decode_step_greedy(want[-1]))
        assert got == want
    tm, _, _ = load_text_model(SimpleNamespace(**base), device="cuda:0")           # (callers from before the flag)
    assert tm.m.kv_cache == "fp8"


def test_speculation_with_the_drafter_head(same_kernels_for_every_row_count):
    """The head's cache is 4-bit too and stays in step; every emitted token is the best one of a model that is fed the same tokens, up to what
    roundings move: the largest distance between the oracle with bf16 activations and the one in fp32, twice (head-on) for each of two runs."""
    from r4dx_b200.models.hybrid import HybridModel
    from r4dx_b200.models.mtp import MtpDrafter
    from r4dx_b200.ops import kernels as K
    from r4dx_b200.runtime.text_model import LocalTextModel
    cfg, q, oracles = _weights(with_mtp=True)
    ids = torch.randint(0, cfg.vocab_size, (37,), generator=torch.Generator().manual_seed(8)).to(torch.int32)
    main = HybridModel(cfg, q, max_ctx=256, kv_cache="int4")
    drafter = MtpDrafter(main, q)
    assert drafter.head.kv_cache == "int4" and all(t.shape[-1] == 9 * cfg.head_dim for t in drafter.head.kv.values())
    tm = LocalTextModel(main, drafter=drafter)
    out = [tm.prefill(ids.tolist())]
    while len(out) < 20:
        out += tm.decode_step_spec_greedy(out[-1], 3)
    assert drafter.head.pos == main.pos - 1
    fed = torch.cat([ids.long(), torch.tensor(out[:-1])])
    ref, rounded = (o.forward(fed)[0] for o in oracles)
    margin = 4 * float((rounded - ref).abs().max())
    for i, tok in enumerate(out):
        row = ref[len(ids) - 1 + i]
        assert float(row.max() - row[tok]) <= margin, i
    # what the two caches hold: the rows of every committed position, finite and not all zero
    for m in (main, drafter.head):
        pos = torch.arange(m.pos, dtype=torch.int32, device="cuda")
        for pool in m.kv.values():
            for x in K.kv4_read(pool, m.block_table, pos):
                assert bool(x.isfinite().all()) and bool((x != 0).flatten(1).any(1).all())


def test_windows_and_single_steps_beside_each_other(same_kernels_for_every_row_count):
    """The same tokens in windows of eight and one by one.  The first attention layer's rows are the same bits; from its output on the runs differ
    in the last bits of attention and what follows from them, in fewer roundings than the oracle with bf16 activations and the one in fp32."""
    from r4dx_b200.models.hybrid import HybridModel
    from r4dx_b200.ops import kernels as K
    cfg, q, oracles = _weights()
    ids = torch.randint(0, cfg.vocab_size, (40,), generator=torch.Generator().manual_seed(3)).to(torch.int32)
    ref, rounded = (o.forward(ids.long())[0] for o in oracles)
    a, b = (HybridModel(cfg, q, max_ctx=256, kv_cache="int4") for _ in range(2))
    windows, steps = [], []
    for s in range(0, 40, 8):
        a.feed(ids[s:s + 8])
        windows.append(a.logits_rows(8).float().cpu().clone())
        for t in range(s, s + 8):
            b.feed(ids[t:t + 1])
            steps.append(b.logits_rows(1).float().cpu().clone())
    windows, steps = torch.cat(windows), torch.cat(steps)
    assert (windows - steps).norm() <= (rounded - ref).norm()
    first = min(a.kv)
    pos = torch.arange(40, dtype=torch.int32, device="cuda")
    for x, y in zip(K.kv4_read(a.kv[first], a.block_table, pos), K.kv4_read(b.kv[first], b.block_table, pos)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("D,Hq,Hkv,rot,norm,gate,T", [(256, 24, 4, 64, True, True, 9), (128, 8, 8, 128, False, False, 33), (64, 32, 8, 22, True, False, 5)])
def test_precore_of_rows_of_many_sequences(D, Hq, Hkv, rot, norm, gate, T):
    """One row of each of T sequences, slots in any order: q against 64 bits, rounded to bf16 (2^-8); k within half a step, what the rounding of the
    scale clips (15 * 2^-8 of a step) and bf16's roundings before and after; v the format's bits; padding rows leave the pool alone."""
    from r4dx_b200.ops import kernels as K
    g = torch.Generator().manual_seed(T)
    theta, qs = 1e6, 2 * D if gate else D
    pos = torch.randint(0, 3000, (T,), generator=g).to(torch.int32)
    pos[T // 2] = -1
    slot = torch.randperm(T, generator=g).to(torch.int32)
    tables = torch.full((T, 3000 // 16 + 1), -1, dtype=torch.int32)
    tables[slot.long(), pos.clamp(min=0).long() // 16] = torch.randperm(T, generator=g).to(torch.int32)
    qg, k, v = torch.randn(T, Hq, qs, generator=g).to(BF), torch.randn(T, Hkv, D, generator=g).to(BF), torch.randn(T, Hkv, D, generator=g).to(BF)
    qn, kn = ((0.1 * torch.randn(D, generator=g)).to(BF) for _ in range(2)) if norm else (None, None)
    cache = torch.full(kv4.pool_shape(T, Hkv, D), 0xFF, dtype=torch.uint8, device="cuda")
    q = torch.full((T, Hq, D), float("nan"), dtype=BF, device="cuda")
    dev = lambda x: None if x is None else x.cuda()  # noqa: E731
    K.attn_precore_kv4(qg.cuda(), k.cuda(), v.cuda(), dev(qn), dev(kn), pos.cuda(), tables.cuda(), q, cache, T, Hq, Hkv, D, rot, theta, q_stride=qs,
                       row_slot=slot.cuda())

    def turned(x, w):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * (1 + w.double())
        h = rot // 2
        a = pos.double()[:, None] * theta ** (-2.0 * torch.arange(h, dtype=torch.float64) / rot)
        c, s = a.cos()[:, None], a.sin()[:, None]
        return torch.cat([x[..., :h] * c - x[..., h:rot] * s, x[..., h:rot] * c + x[..., :h] * s, x[..., rot:]], -1)

    there = pos >= 0
    want = turned(qg[..., :D], qn)
    assert ((q.double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-6)[there].all()
    rk, rv = K.kv4_read(cache, tables.cuda(), pos.cuda(), row_slot=slot.cuda())
    assert torch.equal(rv.cpu()[there], kv4.round_trip(v).to(BF)[there]) and rv[~there.cuda()].isnan().all()
    want = turned(k, kn)
    step = ((want.unflatten(-1, (-1, 64)).amax(-1) - want.unflatten(-1, (-1, 64)).amin(-1)) / 15).repeat_interleave(64, -1)
    bound = (0.5 + 15 * 2.0 ** -8) * 1.01 * step + 2 * 2.0 ** -8 * (want.abs() + step)
    assert ((rk.double().cpu() - want).abs() <= bound)[there].all()
    unused = tables[slot.long()[T // 2], 0]          # the block of the padding row
    assert (cache[int(unused)] == 0xFF).all()
