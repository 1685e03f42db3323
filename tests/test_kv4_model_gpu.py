"""Models with a 4-bit KV cache against the fp32 CPU oracle that rounds keys and values the same way (needs a B200)."""
import pytest
import torch

from r4dx_b200.config import tiny_gemma_config, tiny_hybrid_config, tiny_lfm2_config, tiny_llama_config

pytestmark = pytest.mark.gpu
BF = torch.bfloat16

# How far apart two correct runs are: bf16 activations differ from the oracle's fp32 by 2^-8 at each rounding, and where that moves a key or
# value past a border, its 4-bit code moves by a step, a third of the values' deviation.  The oracle itself, with its activations rounded
# to bf16 where the models round theirs, is 0.026 (hybrid) to 0.106 (short-conv MoE, whose routing flips too) of the logits' norm from the
# oracle in fp32, no kernel being involved.  A model's error is another draw of the same: within twice that, per family, in the 2-norm.
def far(got, ref, rounded):
    return float((got - ref).norm() / ref.norm()), 2 * float((rounded - ref).norm() / ref.norm())


def _family(make):
    from r4dx_b200.models.oracle import OracleModel, init_weights
    from r4dx_b200.quant.weights import dequantize_weight_set, quantize_weight_set
    cfg = make()
    q = quantize_weight_set(cfg, init_weights(cfg, 0))
    dq = dequantize_weight_set(q)
    return (cfg, {k: (v.to("cuda") if hasattr(v, "to") else v) for k, v in q.items()},
            [OracleModel(cfg, dq, int4_kv=True, act_dtype=t) for t in (None, BF)])


@pytest.fixture(scope="module")
def tiny():
    return _family(tiny_hybrid_config)


@pytest.mark.parametrize("make", [tiny_hybrid_config, tiny_llama_config, tiny_gemma_config, tiny_lfm2_config])
def test_small_batches_and_chunks_match_the_oracle(make):
    """Rows eight at a time (decode kernel) and in chunks (prefill kernel), for gated, plain, windowed and short-conv families."""
    from r4dx_b200.models.hybrid import HybridModel
    cfg, q, oracles = _family(make)
    ids = torch.randint(0, cfg.vocab_size, (72,), generator=torch.Generator().manual_seed(1))
    ref, rounded = (o.forward(ids)[0] for o in oracles)
    m = HybridModel(cfg, q, max_ctx=256, kv_cache="int4")
    rows = []
    for s in range(0, 72, 8):
        m.feed(ids[s:s + 8].to(torch.int32))
        rows.append(m.logits_rows(8).float().cpu().clone())
    off, most = far(torch.cat(rows), ref, rounded)
    assert off < most
    c = HybridModel(cfg, q, max_ctx=256, kv_cache="int4")
    c.prefill(ids.to(torch.int32), chunk=40)
    off, _ = far(c.logits_rows(1)[0].float().cpu(), ref[-1], rounded[-1])
    assert off < most
    assert m.state_digest().keys() == c.state_digest().keys()


def test_graph_decode_equals_eager_decode_and_the_cache_is_smaller(tiny):
    from r4dx_b200.models.hybrid import HybridModel
    cfg, q, _ = tiny
    ids = torch.randint(0, cfg.vocab_size, (19,), generator=torch.Generator().manual_seed(2)).to(torch.int32)
    a, b = (HybridModel(cfg, q, max_ctx=256, kv_cache="int4") for _ in range(2))
    assert a.generate_greedy(ids, 40, use_graph=False) == b.generate_greedy(ids, 40, use_graph=True)
    da, db = a.state_digest(), b.state_digest()
    assert all(da[k] == db[k] for k in da if k.startswith("kv."))
    first = b.generate_greedy(ids, 1, use_graph=False)          # (a model that has run goes on; one that is reset begins again)
    a.reset()
    c = HybridModel(cfg, q, max_ctx=256, kv_cache="int4")
    assert len(first) == 1 and a.generate_greedy(ids, 12, use_graph=False) == c.generate_greedy(ids, 12, use_graph=True)
    fp8 = HybridModel(cfg, q, max_ctx=256)
    assert sum(t.numel() for t in a.kv.values()) * 16 == sum(t.numel() for t in fp8.kv.values()) * 9


def test_speculative_windows_continue_like_single_steps(tiny):
    """The last row after windows of eight rows, and after single steps."""
    from r4dx_b200.models.hybrid import HybridModel
    cfg, q, oracles = tiny
    ids = torch.randint(0, cfg.vocab_size, (33,), generator=torch.Generator().manual_seed(3)).to(torch.int32)
    ref, rounded = (o.forward(ids[:32].long())[0] for o in oracles)
    a, b = (HybridModel(cfg, q, max_ctx=256, kv_cache="int4") for _ in range(2))
    for s in range(0, 32, 8):
        a.feed(ids[s:s + 8])
    for s in range(32):
        b.feed(ids[s:s + 1])
    _, most = far(rounded, ref, rounded)
    for m, r in ((a, 7), (b, 0)):
        assert far(m.logits_rows(r + 1)[r].float().cpu(), ref[-1], rounded[-1])[0] < most


def test_batched_decode_matches_the_oracle(tiny):
    """Three slots with prompts of different lengths, one of them given back and taken again."""
    from r4dx_b200.models.batch import BatchModel
    cfg, q, oracles = tiny
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist() for n in (5, 30, 17)]
    bm = BatchModel(cfg, q, slots=4, slot_ctx=128, kv_cache="int4")
    bm.import_slot(1, prompts[0])
    bm.release_slot(1)
    toks = {s: bm.import_slot(s, p) for s, p in zip((2, 1, 3), prompts)}
    got = {s: [t] for s, t in toks.items()}
    logits = {}
    for _ in range(6):
        order = [1, 3, 2]
        nxt = bm.decode_batch(order, [got[s][-1] for s in order])
        for r, s in enumerate(order):
            got[s].append(nxt[r])
            logits.setdefault(s, []).append(bm.last_logits[r].float().cpu())
    for s, p in zip((2, 1, 3), prompts):
        ids = torch.tensor(p + got[s][:-1])
        ref, rounded = (o.forward(ids)[0][len(p):] for o in oracles)
        off, most = far(torch.stack(logits[s]), ref, rounded)
        assert off < most, s


def test_refusals(tiny):
    import dataclasses
    from r4dx_b200.models.hybrid import HybridModel
    cfg, q, _ = tiny
    with pytest.raises(ValueError):
        HybridModel(cfg, q, max_ctx=64, kv_cache="int3")
    with pytest.raises(ValueError):
        HybridModel(dataclasses.replace(cfg, head_dim=96), q, max_ctx=64, kv_cache="int4")
