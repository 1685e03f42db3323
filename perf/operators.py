"""Operators of the 4-bit paged KV cache, as a serving program calls them: rows quantised into the cache (with the norms and the
rotation of q and k before it), rows read back, attention of single tokens, speculative windows and batches over the cache, and
attention of prompt chunks.

The cache.  A pool of blocks of 16 tokens, uint8 [blocks, kv heads, 2 (keys, values), 9 D], head dimension D of 64, 128 or 256.
Every 64 channels of a row are a group with a scale s and a low end lo, both bf16, and codes n of 4 bits: a value is n s + lo.
One block of one head begins with its code words (32 bits: the codes of eight consecutive channels, the first in the lowest
bits), in an order that suits the kernels (`word_places`); then follow the pairs (s, lo) as [token][group].  A block table names
the blocks of a sequence in order.

Head counts are those of the repository's own configurations.
"""
import math

import torch

own = False

BLOCK, GROUP, LIMIT = 16, 64, 32768.0

# query heads, kv heads, head dimension, rotated channels, per-head norm, output gate, rope base
HEADS = {
    "dense": (24, 4, 256, 64, True, True, 1.0e7),
    "moe": (16, 2, 256, 64, True, True, 1.0e7),
    "small": (8, 2, 256, 64, True, True, 1.0e7),
    "llama": (32, 8, 128, 128, False, False, 5.0e5),
    "gemma": (16, 8, 256, 256, True, False, 1.0e6),
    "lfm2": (32, 8, 64, 64, True, False, 1.0e6),
}


def listed():
    return [
        # one decoded token of the dense model after an 8k prompt: its row enters the cache; host calls are what it is made of
        {"name": "write_1", "op": "write", "heads": "dense", "rows": 1, "start": 8191, "batch": False},
        # the headline prompt in one chunk
        {"name": "write_8k", "op": "write", "heads": "dense", "rows": 8192, "start": 0, "batch": False},
        # a few pages of a short conversation inspected, beginning and ending inside a block
        {"name": "read_1k", "op": "read", "heads": "small", "rows": 1003, "start": 5, "batch": False},
        # a long document's cache brought back to 16 bits (ragged)
        {"name": "read_32k", "op": "read", "heads": "llama", "rows": 32517, "start": 0, "batch": False},
        # a reply's token at the start of a conversation, small model
        {"name": "decode_100", "op": "decode", "heads": "small", "rows": 1, "start": 100, "window": 0, "batch": False},
        # the headline: a reply's token after an 8k prompt, dense model
        {"name": "decode_8k", "op": "decode", "heads": "dense", "rows": 1, "start": 8192, "window": 0, "batch": False},
        # a speculative window of one anchor and three drafts, ragged context
        {"name": "window_4", "op": "decode", "heads": "dense", "rows": 4, "start": 12005, "window": 0, "batch": False},
        # a reply deep in a very long document: the cache is what is read
        {"name": "decode_128k", "op": "decode", "heads": "llama", "rows": 1, "start": 131071, "window": 0, "batch": False},
        # a server's step for 48 users, each at a context of its own (up to this length)
        {"name": "batch_48", "op": "decode", "heads": "lfm2", "rows": 48, "start": 6000, "window": 0, "batch": True},
        # a chat turn's prompt of a few hundred tokens
        {"name": "prompt_333", "op": "prefill", "heads": "dense", "rows": 333, "start": 0, "window": 0, "batch": False},
        # a chunk deep in a long document: attention over the earlier chunks
        {"name": "prompt_29k", "op": "prefill", "heads": "dense", "rows": 1024, "start": 29000, "window": 0, "batch": False},
        # a prompt chunk of a sliding-window layer
        {"name": "prompt_window", "op": "prefill", "heads": "gemma", "rows": 4101, "start": 2050, "window": 1024, "batch": False},
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["write", "read", "decode", "prefill"])
    heads = rng.choice(sorted(HEADS))
    hq, hkv, d = HEADS[heads][:3]
    window = rng.choice([0, spread(16, 4096)]) if op in ("decode", "prefill") else 0
    batch = op in ("write", "decode") and rng.random() < 0.4
    if op == "write":
        rows = spread(1, 96) if batch else spread(1, 8192)
        return {"op": op, "heads": heads, "rows": rows, "start": spread(1, 2000 if batch else 30000) - 1, "batch": batch}
    if op == "read":
        return {"op": op, "heads": heads, "rows": spread(1, 32517 * 8 * 128 // (hkv * d)), "start": spread(1, 300) - 1, "batch": False}
    if op == "decode":
        most = 131072 * 8 * 128 // (hkv * d)
        rows = spread(1, 64) if batch else rng.choice([1, 1, rng.randint(2, 8)])
        return {"op": op, "heads": heads, "rows": rows, "start": spread(1, most // rows if batch else most) - 1, "window": window, "batch": batch}
    rows = spread(9, 4096)
    most = 1024 * 29512 * 24 * 256 // (hq * d)          # products of a query head's row and a key, at most the listed case's
    return {"op": op, "heads": heads, "rows": rows, "start": spread(1, max(2, min(29000, most // rows - rows))) - 1, "window": window,
            "batch": False}


def lengths(case):
    """Tokens that each sequence holds after the call."""
    if case["batch"]:      # contexts of all lengths up to the longest, one of them a single token
        n = case["rows"]
        return [1 + case["start"] * i // (n - 1) for i in range(n)] if n > 1 else [1 + case["start"]]
    return [case["start"] + case["rows"]]


# ---- the cache's format, in elementary operations ---------------------------------------------------------------------------------
def word_places(d, values, device):
    """[16, D / 8]: where in a block's code words the word of channels 8 w .. 8 w + 7 of a token lies."""
    t = torch.arange(BLOCK, device=device)[:, None]
    w = torch.arange(d // 8, device=device)[None, :]
    if values:
        g, j, p = w & 7, w >> 3, t >> 1
        if d == 256:
            return t * 32 + (g ^ (t & 6)) * 4 + j
        if d == 128:
            return p * 32 + (g ^ (2 * p & 6)) * 4 + (t & 1) * 2 + j
        return p * 16 + (g ^ ((p & 2) << 1)) * 2 + (t & 1)
    c, j = w & 3, w >> 2
    if d == 256:
        return t * 32 + ((j >> 2) ^ (t & 1)) * 16 + c * 4 + (j & 3)
    return t * (d // 8) + c * (d // 32) + j


def quantise(x):
    """bf16 rows [..., D] -> codes [..., D / 64, 64] (int32), scale and low end [..., D / 64] (fp32 values of bf16)."""
    g = x.float().clamp(-LIMIT, LIMIT).unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1), g.amax(-1)
    s = ((hi - lo) / 15.0).bfloat16().float()
    n = torch.where(s[..., None] > 0, ((g - lo[..., None]) / s[..., None]).round().clamp(0, 15), 8.0)
    return n.to(torch.int32), s, lo


def words_of(n):
    """codes [..., D / 64, 64] -> 32-bit words [..., D / 8]."""
    shift = 4 * torch.arange(8, device=n.device)
    w = (n.flatten(-2).unflatten(-1, (-1, 8)).long() << shift).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


def pairs_of(s, lo):
    return torch.stack([s.bfloat16(), lo.bfloat16()], -1).view(torch.int32)[..., 0]


def put(cache, part, d, block, tok, x):
    """Writes bf16 rows [rows, heads, D] at (block, token of the block) of every head."""
    n, s, lo = quantise(x)
    c32 = cache.view(torch.int32)[:, :, part]                       # [blocks, heads, 9 D / 4]
    head = torch.arange(x.shape[1], device=x.device)[None, :, None]
    at = word_places(d, part == 1, x.device)[tok]                    # [rows, D / 8]
    c32[block[:, None, None], head, at[:, None, :]] = words_of(n)
    pair = 2 * d + tok[:, None] * (d // GROUP) + torch.arange(d // GROUP, device=x.device)
    c32[block[:, None, None], head, pair[:, None, :]] = pairs_of(s, lo)


def get_rows(cache, part, d, block, tok):
    """fp32 values [rows, heads, D] at (block, token of the block) of every head."""
    c32 = cache.view(torch.int32)[:, :, part]
    head = torch.arange(c32.shape[1], device=cache.device)[None, :, None]
    w = c32[block[:, None, None], head, word_places(d, part == 1, cache.device)[tok][:, None, :]]
    n = (w[..., None] >> (4 * torch.arange(8, dtype=torch.int32, device=cache.device))) & 15
    at = 2 * d + tok[:, None] * (d // GROUP) + torch.arange(d // GROUP, device=cache.device)
    pair = c32[block[:, None, None], head, at[:, None, :]].view(torch.bfloat16).float().unflatten(-1, (d // GROUP, 2))
    return (n.flatten(-2).unflatten(-1, (-1, GROUP)) * pair[..., 0:1] + pair[..., 1:2]).flatten(-2)


def get(cache, part, d, blocks):
    """fp32 values [len(blocks) * 16, heads, D] of whole blocks."""
    c32 = cache.view(torch.int32)[:, :, part][blocks]               # [n, heads, 9 D / 4]
    w = c32[..., :2 * d][..., word_places(d, part == 1, cache.device)]          # [n, heads, 16, D / 8]
    n = (w[..., None] >> (4 * torch.arange(8, dtype=torch.int32, device=cache.device))) & 15
    pair = c32[..., 2 * d:].contiguous().view(torch.bfloat16).float().unflatten(-1, (BLOCK, d // GROUP, 2))
    x = n.flatten(-2).unflatten(-1, (-1, GROUP)) * pair[..., 0:1] + pair[..., 1:2]
    return x.flatten(-2).permute(0, 2, 1, 3).flatten(0, 1)


# ---- inputs -------------------------------------------------------------------------------------------------------------------
def content(case, seed, device):
    """Rows that the cache holds, one sequence after another: keys (with the channels of large amplitude and the offsets that keys
    have) and values, bf16 [tokens, heads, D]."""
    hq, hkv, d = HEADS[case["heads"]][:3]
    g = torch.Generator(device=device).manual_seed(seed * 7919 + 11)
    held = sum(lengths(case))
    loud = 0.6 * torch.exp(0.5 * torch.randn(1, hkv, d, generator=g, device=device))
    off = 0.3 * torch.randn(1, hkv, d, generator=g, device=device)
    k = (torch.randn(held, hkv, d, generator=g, device=device) * loud + off).bfloat16()
    v = (torch.randn(held, hkv, d, generator=g, device=device) * 0.5).bfloat16()
    return k, v


def prepare(case, seed):
    dev = "cuda"
    hq, hkv, d, rot, norm, gate, theta = HEADS[case["heads"]]
    seqs = lengths(case)
    need = [(n + BLOCK - 1) // BLOCK for n in seqs]
    g = torch.Generator(device=dev).manual_seed(seed * 104729 + 5)
    pool = sum(need) + 3
    order = torch.randperm(pool, generator=g, device=dev).to(torch.int32)
    table = torch.zeros(len(seqs), max(need) + 1, dtype=torch.int32, device=dev)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    cache = torch.zeros(pool, hkv, 2, 9 * d, dtype=torch.uint8, device=dev)
    rows = case["rows"]
    s = {"case": dict(case), "cache": cache, "table": table if case["batch"] else table[0].contiguous(),
         "slot": torch.arange(rows, dtype=torch.int32, device=dev).flip(0).contiguous() if case["batch"] else None}
    if case["batch"]:      # one row of each sequence, the last token
        s["pos"] = torch.tensor([n - 1 for n in seqs], dtype=torch.int32, device=dev)[s["slot"].long()]
    else:
        s["pos"] = torch.arange(case["start"], case["start"] + rows, dtype=torch.int32, device=dev)
    k, v = content(case, seed, dev)
    if case["op"] == "write":
        e = lambda *shape: torch.randn(*shape, generator=g, device=dev)  # noqa: E731
        s["qg"] = e(rows, hq, 2 * d if gate else d).bfloat16()
        s["k"], s["v"] = k[-rows:].contiguous(), v[-rows:].contiguous()
        s["qn"], s["kn"] = ((0.1 * e(d)).bfloat16(), (0.1 * e(d)).bfloat16()) if norm else (None, None)
        s["q"] = torch.empty(rows, hq, d, dtype=torch.bfloat16, device=dev)
        return s
    seq = torch.repeat_interleave(torch.arange(len(seqs), device=dev), torch.tensor(seqs, device=dev))
    tok = torch.cat([torch.arange(n, device=dev) for n in seqs])
    block = table[seq, tok // BLOCK].long()
    put(cache, 0, d, block, tok % BLOCK, k)
    put(cache, 1, d, block, tok % BLOCK, v)
    if case["op"] == "read":
        s["k"] = torch.empty(rows, hkv, d, dtype=torch.bfloat16, device=dev)
        s["v"] = torch.empty(rows, hkv, d, dtype=torch.bfloat16, device=dev)
        return s
    s["q"] = (1.5 * torch.randn(rows, hq, d, generator=g, device=dev)).bfloat16()
    s["qg"] = torch.randn(rows, hq, 2 * d, generator=g, device=dev).bfloat16() if gate else None
    s["out"] = torch.empty(rows, hq, d, dtype=torch.bfloat16, device=dev)
    return s


# ---- the operators, plain ---------------------------------------------------------------------------------------------------------
def rotated(x, pos, rot, theta):
    """The first `rot` channels of fp32 [rows, heads, D] turned by their positions' angles (halves as pairs), angles in 64 bits."""
    i = torch.arange(rot // 2, dtype=torch.float64, device=x.device)
    a = pos.double()[:, None] * (float(theta) ** (-2.0 * i / rot))
    c, s = a.cos().float()[:, None], a.sin().float()[:, None]
    x1, x2 = x[..., :rot // 2], x[..., rot // 2:rot]
    return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s, x[..., rot:]], -1)


def normed(x, w):
    return x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * (1.0 + w.float())


def write(s):
    hq, hkv, d, rot, norm, gate, theta = HEADS[s["case"]["heads"]]
    pos = s["pos"]
    table = s["table"][s["slot"].long()] if s["case"]["batch"] else s["table"][None].expand(pos.shape[0], -1)
    block = table.gather(1, pos.long()[:, None] // BLOCK)[:, 0].long()
    tok = pos.long() % BLOCK
    q = rotated(normed(s["qg"][..., :d].float(), s["qn"]), pos, rot, theta).bfloat16()
    k = rotated(normed(s["k"].float(), s["kn"]), pos, rot, theta).bfloat16()
    put(s["cache"], 0, d, block, tok, k)
    put(s["cache"], 1, d, block, tok, s["v"])
    return {"q": q, "k": get_rows(s["cache"], 0, d, block, tok).bfloat16(), "v": get_rows(s["cache"], 1, d, block, tok).bfloat16()}


def read(s):
    d, first, n = HEADS[s["case"]["heads"]][2], s["case"]["start"], s["case"]["rows"]
    blocks = s["table"][first // BLOCK:(first + n + BLOCK - 1) // BLOCK].long()
    skip = first % BLOCK
    return {"k": get(s["cache"], 0, d, blocks)[skip:skip + n].bfloat16(), "v": get(s["cache"], 1, d, blocks)[skip:skip + n].bfloat16()}


def attend(q, k, v, pos, kpos, window):
    """fp32 rows [..., rows, heads, D] against keys [..., keys, kv heads, D]: softmax over the keys at or before each row's position."""
    hq, hkv, d = q.shape[-2], k.shape[-2], q.shape[-1]
    q = q.unflatten(-2, (hkv, hq // hkv)).movedim(-4, -2).flatten(-3, -2)       # [..., kv heads, group * rows, D]
    scores = (q @ k.movedim(-2, -3).mT) * d ** -0.5
    seen = kpos[..., None, :] <= pos[..., :, None]
    if window:
        seen = seen & (kpos[..., None, :] > pos[..., :, None] - window)
    rows = pos.shape[-1]
    scores = scores.unflatten(-2, (-1, rows)).masked_fill_(~seen[..., None, None, :, :], float("-inf"))
    p = torch.exp_(scores - scores.amax(-1, keepdim=True))
    o = (p / p.sum(-1, keepdim=True)).flatten(-3, -2) @ v.movedim(-2, -3)       # [..., kv heads, group * rows, D]
    return o.unflatten(-2, (-1, rows)).movedim(-2, -4).flatten(-3, -2)


def attention(s):
    case = s["case"]
    d = HEADS[case["heads"]][2]
    pos = s["pos"]
    if case["batch"]:      # every sequence padded to the longest
        used = (case["start"] + 1 + BLOCK - 1) // BLOCK
        blocks = s["table"][s["slot"].long(), :used].long()
        k, v = (get(s["cache"], part, d, blocks.flatten()).unflatten(0, (case["rows"], -1)) for part in (0, 1))
        kpos = torch.arange(k.shape[1], device=k.device).expand(case["rows"], -1)
        o = attend(s["q"].float()[:, None], k, v, pos[:, None], kpos, case["window"])[:, 0]
    else:
        end = case["start"] + case["rows"]
        first = max(0, case["start"] - case["window"] + 1) // BLOCK if case["window"] else 0
        blocks = s["table"][first:(end + BLOCK - 1) // BLOCK].long()
        k, v = get(s["cache"], 0, d, blocks), get(s["cache"], 1, d, blocks)
        o = attend(s["q"].float(), k, v, pos, first * BLOCK + torch.arange(k.shape[0], device=k.device), case["window"])
    return {"out": (o if s["qg"] is None else o * torch.sigmoid(s["qg"][..., d:].float())).bfloat16()}


def run(s):
    case = s["case"]
    if not own:
        return {"write": write, "read": read, "decode": attention, "prefill": attention}[case["op"]](s)
    from r4dx_b200.ops import kernels as K
    hq, hkv, d, rot, norm, gate, theta = HEADS[case["heads"]]
    if case["op"] == "write":
        K.attn_precore_kv4(s["qg"], s["k"], s["v"], s["qn"], s["kn"], s["pos"], s["table"], s["q"], s["cache"], case["rows"], hq, hkv, d, rot,
                           theta, q_stride=2 * d if gate else d, row_slot=s["slot"])
        k, v = K.kv4_read(s["cache"], s["table"], s["pos"], row_slot=s["slot"])
        return {"q": s["q"], "k": k, "v": v}
    if case["op"] == "read":
        K.kv4_read(s["cache"], s["table"], s["pos"], s["k"], s["v"])
        return {"k": s["k"], "v": s["v"]}
    if case["op"] == "decode":
        K.attn_decode_kv4(s["q"], s["qg"], s["cache"], s["table"], s["pos"], s["out"], case["rows"], hq, hkv, d, gated=gate,
                          window=case["window"], row_slot=s["slot"])
    else:
        K.attn_prefill_kv4(s["q"], s["qg"], s["cache"], s["table"], s["out"], case["rows"], hq, hkv, d, case["start"], gated=gate,
                           window=case["window"])
    return {"out": s["out"]}


def work(case):
    hq, hkv, d, rot, norm, gate, theta = HEADS[case["heads"]]
    rows, held = case["rows"], 2 * hkv * d * 9 // 16            # bytes of a token in the cache
    if case["op"] == "write":      # q in and out, k and v in, the cache's rows out and the values they stand for
        return {"bytes": rows * (4 * hq * d + 4 * hkv * d + held + 4 * hkv * d), "flops": rows * (8 * (hq + hkv) * d + 8 * hkv * d)}
    if case["op"] == "read":
        return {"bytes": rows * (held + 4 * hkv * d), "flops": rows * 4 * hkv * d}
    if case["batch"]:
        keys = pairs = sum(min(n, case["window"] or n) for n in lengths(case))
    else:
        end, w = case["start"] + rows, case["window"]
        keys = end - (max(0, case["start"] - w + 1) if w else 0)
        pairs = sum(min(p + 1, w or p + 1) for p in range(case["start"], end))
    return {"bytes": keys * held + rows * hq * d * (6 if gate else 4), "flops": 4 * pairs * hq * d}


# ---- the same in 64 bits, from the definition ---------------------------------------------------------------------------------------
def exact(case, seed):
    dev = "cuda"
    hq, hkv, d, rot, norm, gate, theta = HEADS[case["heads"]]
    s = prepare(case, seed)
    k, v = content(case, seed, dev)
    rows = case["rows"]

    def stands_for(x):      # what the codes of bf16 rows stand for, group by group
        out = torch.empty(x.shape, dtype=torch.float64, device=dev)
        for a in range(0, d, GROUP):
            g = x[..., a:a + GROUP].double().clamp(-LIMIT, LIMIT)
            lo = g.min(-1, keepdim=True).values
            step = ((g.max(-1, keepdim=True).values - lo).float() / 15).bfloat16().double()
            n = torch.round((g - lo) / step).clamp(0, 15)
            out[..., a:a + GROUP] = torch.where(step > 0, n * step + lo, lo)
        return out

    if case["op"] == "write":
        def turned(x, w):
            x = x.double()
            if w is not None:
                x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * (1 + w.double())
            y = x.clone()
            for i in range(rot // 2):
                a = s["pos"].double() * math.exp(-math.log(theta) * 2 * i / rot)
                c, n = torch.cos(a)[:, None], torch.sin(a)[:, None]
                y[..., i] = x[..., i] * c - x[..., i + rot // 2] * n
                y[..., i + rot // 2] = x[..., i + rot // 2] * c + x[..., i] * n
            return y
        return {"q": turned(s["qg"][..., :d], s["qn"]), "k": stands_for(turned(s["k"], s["kn"]).bfloat16()), "v": stands_for(s["v"])}
    if case["op"] == "read":
        return {"k": stands_for(k[case["start"]:]), "v": stands_for(v[case["start"]:])}
    out = torch.empty(rows, hq, d, dtype=torch.float64, device=dev)
    seqs = lengths(case)
    starts = [sum(seqs[:i]) for i in range(len(seqs))]
    slots = s["slot"].tolist() if case["batch"] else [0]
    for i, slot in enumerate(slots):
        at = slice(i, i + 1) if case["batch"] else slice(0, rows)
        pos = s["pos"][at].double()
        for h in range(hkv):
            own_k = stands_for(k[starts[slot]:starts[slot] + seqs[slot], h])
            own_v = stands_for(v[starts[slot]:starts[slot] + seqs[slot], h])
            kp = torch.arange(seqs[slot], dtype=torch.float64, device=dev)
            hidden = kp[None] > pos[:, None]
            if case["window"]:
                hidden = hidden | (kp[None] <= pos[:, None] - case["window"])
            for a in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                logits = s["q"][at, a].double() @ own_k.T / math.sqrt(d)
                out[at, a] = torch.softmax(logits.masked_fill(hidden, -math.inf), -1) @ own_v
    return {"out": out if s["qg"] is None else out / (1 + torch.exp(-s["qg"][..., d:].double()))}
