"""GPU model graph of the Qwen-style hybrid decoder (dense), single rank or one TP rank.

PyTorch is the framework layer here: module wiring, state allocation (paged fp8 or 4-bit KV, GDN state,
conv ring), workspaces and CUDA-graph capture.  Every op on the token path is a kernel of
``libr4dxb_cuda.so``.  The forward follows the reference's chunk pipeline -- prologue (ids ->
embedding), layer range, epilogue (final norm, LM head, argmax)
(reference: src/model/model.cpp:1228-1935) -- but state handling is designed for replayable
graphs: positions, the committed-row count and the token feedback all live in device memory.
"""
from __future__ import annotations

import os

import math
from dataclasses import dataclass
from typing import Callable, Dict, List, Optional

import torch

from ..config import ModelConfig
from ..ops import kernels as K
from ..quant.kv4 import HEAD_DIMS
from ..quant.trellis import TrellisWeight
from ..quant.w4a16 import W4Weight, W8Weight

BF = torch.bfloat16
MAX_ROWS = 8          # rows per small-batch call (decode = 1, verify window <= 8)
KV_BLOCK = 16
CONV_RING = 16


class Linear:
    """One weight in whatever layout the container gave it; y = x W^T for T <= MAX_ROWS rows."""

    def __init__(self, w, name: str = ""):
        self.w = w
        self.name = name
        if isinstance(w, TrellisWeight):
            self.N, self.K = w.N, w.K
            self.ksplit = K.pick_ksplit(w.N, w.K)
        elif isinstance(w, (W4Weight, W8Weight)):
            self.N, self.K = w.N, w.K
        else:
            self.N, self.K = w.shape

    def __call__(self, x: torch.Tensor, out: torch.Tensor, residual: Optional[torch.Tensor] = None,
                 prologue: int = 0, norm_w: Optional[torch.Tensor] = None, eps: float = 1e-6) -> torch.Tensor:
        w = self.w
        if isinstance(w, TrellisWeight):
            T = x.numel() // (2 * self.K if prologue in (K.PRO_SILU_MUL, K.PRO_GELU_MUL) else self.K)
            return K.trellis_gemv(w, x, residual=residual, out=out, ksplit=self.ksplit, prologue=prologue,
                                  norm_w=norm_w, eps=eps, split_rows=K.rows_split(self.N, self.K, T))
        if isinstance(w, (W4Weight, W8Weight)):
            # group-quantised layouts: the streaming kernels have no prologue / residual modes, so the producer of the
            # activations and the residual add are kernels of their own (the w8a16 body of the dense and short-conv
            # families; reference: docs/w8a16.md)
            xin = x
            if prologue == K.PRO_RMSNORM:
                xin = K.rmsnorm(x, norm_w, eps)           # containers hold every norm weight in the (1 + w) convention
            elif prologue == K.PRO_SILU_MUL:
                xin = K.silu_mul(x)
            elif prologue == K.PRO_GELU_MUL:
                raise NotImplementedError("GeGLU with a group-quantised down projection")
            gemv = K.w8a16_gemv if isinstance(w, W8Weight) else K.w4a16_gemv
            if residual is None:
                return gemv(w, xin, out_f32=(out.dtype == torch.float32), out=out)
            tmp = gemv(w, xin, out_f32=False)
            if residual.data_ptr() != out.data_ptr():
                out.copy_(residual)
            return K.residual_add(out, tmp)
        raise NotImplementedError(f"layout of {self.name}")

    def many(self, x: torch.Tensor, out: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
             out_f32: bool = False) -> torch.Tensor:
        """Any number of rows of a w4a16 or dense weight on the tensor cores (no input transform in these layouts)."""
        w = self.w
        if isinstance(w, TrellisWeight):
            raise NotImplementedError(f"{self.name}: trellis weights take chunk() for many rows")
        if out is not None:
            out_f32 = out.dtype == torch.float32
        return K.linear_tc(w, x, residual=residual, out=out, out_f32=out_f32)

    def chunk(self, x: torch.Tensor, xh_buf: torch.Tensor, out: torch.Tensor, residual: Optional[torch.Tensor] = None,
              fused_silu_mul: bool = False, gelu: bool = False) -> torch.Tensor:
        """Large-T path: input transform (optionally fused with SwiGLU) + tcgen05 GEMM."""
        w = self.w
        if isinstance(w, (W4Weight, W8Weight)):
            xin = x
            if fused_silu_mul:
                if gelu:
                    raise NotImplementedError("GeGLU with a group-quantised down projection")
                xin = K.silu_mul(x)
            return K.linear_tc(w, xin, residual=residual, out=out)
        if not isinstance(w, TrellisWeight):
            raise NotImplementedError(f"chunk path for layout of {self.name}")
        T = out.shape[0]
        xh = xh_buf.view(-1)[:T * w.K].view(T, w.K)
        K.trellis_input(x, w.suh, out=xh, fused_silu_mul=fused_silu_mul, gelu=gelu)
        if K.PREFILL_F8 and T >= 128 and w.K % 128 == 0:
            # opt-in 8-bit product: the e4m3 rows and their scales live in the unused tail of the transform buffer
            tail = xh_buf.view(-1)[T * w.K:]
            if tail.numel() * 2 >= T * w.K + 4 * T + 16:
                xq = tail.view(torch.uint8)[:T * w.K].view(T, w.K)
                sc = tail.view(torch.uint8)[(T * w.K + 15) // 16 * 16:][:4 * T].view(torch.float32)
            else:
                xq, sc = None, None
            xq, sc = K.quantize_rows_e4m3(xh, xq, sc)
            return K.trellis_gemm_f8(w, xq, sc, residual=residual, out=out)
        return K.trellis_gemm(w, xh, residual=residual, out=out)

    @property
    def nbytes(self) -> int:
        w = self.w
        return w.nbytes if hasattr(w, "nbytes") and not isinstance(w, torch.Tensor) else w.numel() * w.element_size()


class _NullCtx:
    def __enter__(self):
        return None

    def __exit__(self, *a):
        return False


@dataclass
class StepBuffers:
    """Workspaces for one call of up to MAX_ROWS rows (allocated once; graph-safe)."""
    ids: torch.Tensor
    positions: torch.Tensor
    n_replay: torch.Tensor
    status_and_ids: torch.Tensor     # the GEMM status word as of the latest argmax, then `next_ids`: one read-back brings both
    next_ids: torch.Tensor
    next_vals: torch.Tensor
    x: torch.Tensor
    h: torch.Tensor
    mixed: torch.Tensor
    z: torch.Tensor
    ab: torch.Tensor
    core: torch.Tensor
    qg: torch.Tensor
    k: torch.Tensor
    v: torch.Tensor
    q: torch.Tensor
    gate_up: torch.Tensor
    act: torch.Tensor
    logits: torch.Tensor
    argmax_scratch: torch.Tensor
    part_acc: torch.Tensor
    part_ml: torch.Tensor


class HybridModel:
    def __init__(self, cfg: ModelConfig, weights: Dict[str, object], max_ctx: int = 8192 + 1024,
                 device: str = "cuda", attn_splits: Optional[int] = None, comm=None, layer_range=None, kv_cache: str = "fp8"):
        """``layer_range`` = (first, end): a pipeline stage that runs only those layers (embedding with the
        first stage, head with the last).  ``kv_cache``: "fp8" (e4m3, a static descale per head) or "int4" (4-bit codes with a
        bf16 scale and low end per 64 channels, quant/kv4.py: 9/16 of the bytes, no descales)."""
        cfg.validate() if cfg.tp_world == 1 else None
        if kv_cache not in ("fp8", "int4"):
            raise ValueError(f"kv_cache {kv_cache!r}: fp8 or int4")
        if kv_cache == "int4" and cfg.head_dim not in HEAD_DIMS:
            raise ValueError(f"the 4-bit KV cache has head dimensions {HEAD_DIMS}, not {cfg.head_dim}")
        self.kv_cache = kv_cache
        if cfg.has_conv_layers and comm is not None and comm.world > 1 and os.environ.get("R4DXB_UNVALIDATED_TP") != "1":
            # the sharding of this family is checked on the CPU (shards add up to the unsharded block); its only two-GPU run
            # did not finish within its time limit and the cause has not been found, so the path stays closed by default
            raise NotImplementedError("tensor-parallel execution of the short-conv family is not validated on GPUs yet "
                                      "(set R4DXB_UNVALIDATED_TP=1 to run it anyway)")
        self.cfg = cfg
        self.device = torch.device(device)
        self.comm = comm                       # tensor-parallel communicator (None = single rank)
        self.layer_begin, self.layer_end = layer_range if layer_range is not None else (0, cfg.num_hidden_layers)
        self.max_ctx = ((max_ctx + KV_BLOCK - 1) // KV_BLOCK) * KV_BLOCK
        self.w = weights
        self.lin: Dict[str, Linear] = {}
        for name, t in weights.items():
            if isinstance(t, (TrellisWeight, W4Weight, W8Weight)):
                self.lin[name] = Linear(t, name)
        # fused [a; b] gate projection per GDN layer
        # residual-stream rotation: a weight set that carries it runs its layers in the basis x Q (quant/rotation.py)
        self.rot = None
        if "rotation.signs" in weights and self.layer_begin is not None:
            signs = weights["rotation.signs"].to(self.device, torch.float32).contiguous()
            mix = weights["rotation.mix"].to(self.device, torch.float32).contiguous()
            if signs.numel() != cfg.hidden_size or mix.dim() != 2 or mix.shape[0] != mix.shape[1] or cfg.hidden_size % mix.shape[0]:
                raise ValueError("rotation tensors do not fit the model's hidden size")
            self.rot = (signs, mix)
        self.ab_w: Dict[int, torch.Tensor] = {}
        for i in range(self.layer_begin, self.layer_end):
            if not cfg.is_attention_layer(i) and not cfg.is_conv_layer(i):
                p = f"text.layers.{i}.gdn."
                self.ab_w[i] = torch.cat([weights[p + "in_proj_a"], weights[p + "in_proj_b"]], 0).contiguous()
        self._alloc_state(attn_splits)
        self.moe = {}
        if cfg.is_moe:
            from .moe import MoeBlock
            er = getattr(comm, "expert_range", None) if comm is not None else None
            for i in range(max(self.layer_begin, cfg.num_dense_layers), self.layer_end):
                self.moe[i] = MoeBlock(cfg, weights, i, self.device, MAX_ROWS, *(er or (0, cfg.num_experts)))
        self._graphs: Dict[int, torch.cuda.CUDAGraph] = {}
        self.pos = 0                           # host mirror of the next position
        self.pending_rows = 0                  # rows of the last call not yet committed to the GDN base state

    # ------------------------------------------------------------------------------------------
    def _alloc_state(self, attn_splits: Optional[int]) -> None:
        cfg, dev = self.cfg, self.device
        H = cfg.hidden_size
        Hq, Hkv, D = cfg.num_attention_heads, cfg.num_key_value_heads, cfg.head_dim
        Hv, Hk, Dg = cfg.linear_num_value_heads, cfg.linear_num_key_heads, cfg.linear_key_head_dim
        nblk = self.max_ctx // KV_BLOCK + 1       # one spare block: scratch positions for graph warm-up
        self.block_table = torch.arange(nblk, dtype=torch.int32, device=dev)
        self.kv: Dict[int, torch.Tensor] = {}
        self.gdn_state: Dict[int, torch.Tensor] = {}
        self.ring: Dict[int, torch.Tensor] = {}
        self.log_u: Dict[int, torch.Tensor] = {}
        self.log_k: Dict[int, torch.Tensor] = {}
        self.log_eg: Dict[int, torch.Tensor] = {}
        for i in range(self.layer_begin, self.layer_end):
            if cfg.is_attention_layer(i):
                self.kv[i] = self.new_pool(nblk)
            elif cfg.is_conv_layer(i):
                self.ring[i] = torch.zeros(32, cfg.conv_channels, dtype=BF, device=dev)   # B * x rows keyed by position & 31
            else:
                self.gdn_state[i] = torch.zeros(Hv, Dg, Dg, dtype=torch.float32, device=dev)
                self.ring[i] = torch.zeros(CONV_RING, cfg.conv_dim, dtype=BF, device=dev)
                self.log_u[i] = torch.zeros(MAX_ROWS, Hv, Dg, dtype=torch.float32, device=dev)
                self.log_k[i] = torch.zeros(MAX_ROWS, Hv, Dg, dtype=torch.float32, device=dev)
                self.log_eg[i] = torch.zeros(MAX_ROWS, Hv, dtype=torch.float32, device=dev)
        if attn_splits is None:
            attn_splits = max(1, min(64, (148 + Hkv - 1) // max(1, Hkv)))
        self.attn_splits = attn_splits
        G = (Hq // max(1, Hkv)) * MAX_ROWS
        R = MAX_ROWS
        V = cfg.vocab_shard_size
        e = lambda *s, dtype=BF: torch.zeros(*s, dtype=dtype, device=dev)
        status_and_ids = e(1 + R, dtype=torch.int32)
        self.buf = StepBuffers(
            ids=e(R, dtype=torch.int32), positions=e(R, dtype=torch.int32), n_replay=e(1, dtype=torch.int32),
            status_and_ids=status_and_ids, next_ids=status_and_ids[1:], next_vals=e(R, dtype=torch.float32),
            x=e(R, H), h=e(R, H), mixed=e(R, max(cfg.conv_dim, 3 * H if cfg.has_conv_layers else 0)), z=e(R, cfg.value_dim),
            ab=e(R, 2 * Hv, dtype=torch.float32), core=e(R, max(cfg.value_dim, cfg.q_dim, H if cfg.has_conv_layers else 0)),
            qg=e(R, cfg.q_proj_dim), k=e(R, cfg.kv_dim), v=e(R, cfg.kv_dim), q=e(R, cfg.q_dim),
            gate_up=e(R, 2 * max(cfg.intermediate_size, 1)), act=e(R, max(cfg.intermediate_size, 1)),
            logits=e(R, V, dtype=torch.float32), argmax_scratch=e(2 * R * 256, dtype=torch.float32),
            part_acc=e(attn_splits * Hkv * G * D, dtype=torch.float32),
            part_ml=e(attn_splits * Hkv * G * 2, dtype=torch.float32))
        self.kv4_scratch = None                  # for the rows of a call, whatever their number
        if self.kv_cache == "int4" and self.kv:
            self.kv4_scratch = e(max(1, *(K.kv4_scratch_floats(T, 1, Hq, Hkv, D, nblk) for T in range(1, R + 1))), dtype=torch.float32)

    def new_pool(self, blocks: int) -> torch.Tensor:
        """An empty pool of KV blocks of one layer."""
        Hkv, D = self.cfg.num_key_value_heads, self.cfg.head_dim
        if self.kv_cache == "int4":
            return K.kv4_cache(blocks, Hkv, D, self.device)
        return torch.zeros(blocks, Hkv, 2, KV_BLOCK, D, dtype=torch.uint8, device=self.device)

    # ---- attention over the cache (either format) --------------------------------------------------
    def _attn_write(self, i: int, qg, k, v, positions, q, T: int) -> None:
        """Norms and rope of the rows' queries and keys; keys and values enter layer i's cache."""
        cfg, w, p = self.cfg, self.w, f"text.layers.{i}.attn."
        Hq, Hkv, D = cfg.num_attention_heads, cfg.num_key_value_heads, cfg.head_dim
        if self.kv_cache == "int4":
            K.attn_precore_kv4(qg, k, v, w.get(p + "q_norm"), w.get(p + "k_norm"), positions, self.block_table, q, self.kv[i], T, Hq, Hkv, D,
                               cfg.rotary_dim, cfg.layer_theta(i), cfg.rms_norm_eps, q_stride=cfg.q_proj_dim // Hq)
        else:
            K.attn_precore(qg, k, v, w.get(p + "q_norm"), w.get(p + "k_norm"), w[p + "k_descale"], w[p + "v_descale"], positions,
                           self.block_table, q, self.kv[i], T, Hq, Hkv, D, cfg.rotary_dim, cfg.layer_theta(i), cfg.rms_norm_eps,
                           q_stride=cfg.q_proj_dim // Hq)

    def _attn_rows(self, i: int, T: int, core: torch.Tensor) -> None:
        """Attention of the T staged rows."""
        cfg, b, w, p = self.cfg, self.buf, self.w, f"text.layers.{i}.attn."
        Hq, Hkv, D = cfg.num_attention_heads, cfg.num_key_value_heads, cfg.head_dim
        if self.kv_cache == "int4":
            K.attn_decode_kv4(b.q, b.qg, self.kv[i], self.block_table, b.positions, core, T, Hq, Hkv, D, cfg.attn_output_gate,
                              cfg.layer_window(i), scratch=self.kv4_scratch)
        else:
            K.attn_decode(b.q, b.qg, self.kv[i], self.block_table, b.positions, w[p + "k_descale"], w[p + "v_descale"],
                          b.part_acc, b.part_ml, core, T, Hq, Hkv, D, self.attn_splits, cfg.attn_output_gate,
                          window=cfg.layer_window(i))

    def _attn_chunk(self, i: int, q, qg, core, T: int, pos0: int) -> None:
        """Attention of a prompt chunk's T rows at positions pos0 .."""
        cfg, w, p = self.cfg, self.w, f"text.layers.{i}.attn."
        Hq, Hkv, D, win = cfg.num_attention_heads, cfg.num_key_value_heads, cfg.head_dim, cfg.layer_window(i)
        limit = self._key_limit if win > 0 else None
        if self.kv_cache == "int4":
            K.attn_prefill_kv4(q, qg, self.kv[i], self.block_table, core, T, Hq, Hkv, D, pos0, cfg.attn_output_gate, win, limit)
        else:
            K.attn_prefill(q, qg, self.kv[i], self.block_table, w[p + "k_descale"], w[p + "v_descale"], core, T, Hq, Hkv, D, pos0,
                           cfg.attn_output_gate, window=win, key_limit=limit)

    def state_bytes(self) -> int:
        n = 0
        for d in (self.kv, self.gdn_state, self.ring):
            n += sum(t.numel() * t.element_size() for t in d.values())
        return n

    def weight_bytes(self) -> int:
        n = 0
        for t in self.w.values():
            n += t.nbytes if not isinstance(t, torch.Tensor) else t.numel() * t.element_size()
        return n

    def streamed_bytes_per_token(self) -> int:
        """Bytes every decoded token must read: all quantized linears + the LM head shard."""
        return sum(l.nbytes for l in self.lin.values() if ".experts." not in l.name) + sum(m.nbytes for m in self.moe.values())

    # ------------------------------------------------------------------------------------------
    def reset(self) -> None:
        for d in (self.kv, self.gdn_state, self.ring):
            for t in d.values():
                t.zero_()
        self.buf.n_replay.zero_()
        self.pos = 0
        self.pending_rows = 0

    # ---- sibling overlap ----------------------------------------------------------------------------
    overlap_siblings = os.environ.get("R4DXB_OVERLAP", "1") != "0"

    def _fork(self):
        # measured: +6 % at TP=1 and TP=2; at TP=8 the projections are a few microseconds each and the extra graph
        # edges cost more than the overlap returns (137 vs 150 tok/s), so wide tensor-parallel groups run in line
        if not self.overlap_siblings or (self.comm is not None and self.comm.world >= 4):
            return None
        if getattr(self, "_side", None) is None:
            self._side = torch.cuda.Stream(device=self.device)
        self._side.wait_stream(torch.cuda.current_stream())
        return self._side

    def _join(self, side) -> None:
        if side is not None:
            torch.cuda.current_stream().wait_stream(side)

    # ---- sibling projections in one launch -----------------------------------------------------------
    fuse_siblings = os.environ.get("R4DXB_SIBLINGS", "1") != "0"

    def _siblings(self, names):
        """The one-launch group of these projections, or None when they cannot share a launch (other layouts, unequal
        bit widths) or the switch is off; built once per name tuple."""
        if not self.fuse_siblings:
            return None
        cache = self.__dict__.setdefault("_sibling_groups", {})
        if names not in cache:
            ws = [self.lin[n].w for n in names]
            ok = all(isinstance(w_, TrellisWeight) for w_ in ws) and len({(w_.K, w_.kb) for w_ in ws}) == 1
            cache[names] = K.SiblingGroup(ws) if ok else None
        return cache[names]

    # ---- layers ---------------------------------------------------------------------------------
    def _gdn_layer(self, i: int, T: int) -> None:
        cfg, b, w = self.cfg, self.buf, self.w
        p = f"text.layers.{i}.gdn."
        Hv, Hk, Dg = cfg.linear_num_value_heads, cfg.linear_num_key_heads, cfg.linear_key_head_dim
        x, nw, eps = b.x[:T], w[f"text.layers.{i}.input_layernorm"], cfg.rms_norm_eps
        # the three projections read the same rows and write different buffers: the two small ones run on a side
        # stream (a parallel branch of the captured graph) while the large one fills the machine
        grp = self._siblings((p + "in_proj_qkv", p + "in_proj_z"))
        ab_w = self.ab_w[i] if self.fuse_siblings and self.ab_w[i].shape[0] == 2 * Hv else None   # a / b inside the GDN kernel
        side = self._fork() if (grp is None or ab_w is None) else None
        if grp is not None:
            grp(x, (b.mixed[:T], b.z[:T]), prologue=K.PRO_RMSNORM, norm_w=nw, eps=eps)
        else:
            self.lin[p + "in_proj_qkv"](x, out=b.mixed[:T], prologue=K.PRO_RMSNORM, norm_w=nw, eps=eps)
        with torch.cuda.stream(side) if side is not None else _NullCtx():
            if grp is None:
                self.lin[p + "in_proj_z"](x, out=b.z[:T], prologue=K.PRO_RMSNORM, norm_w=nw, eps=eps)
            if ab_w is None:
                K.bf16_gemv_norm(self.ab_w[i], x, nw, eps, b.ab[:T])
        self._join(side)
        K.gdn_decode(b.mixed, b.z, b.ab, w[p + "conv1d_weight"], w[p + "A_log"], w[p + "dt_bias"], w[p + "norm_weight"],
                     self.ring[i], self.gdn_state[i], self.log_u[i], self.log_k[i], self.log_eg[i], b.positions,
                     b.n_replay, b.core, T, Hv, Hk, Dg, cfg.rms_norm_eps, ab_w=ab_w, x=x, in_norm_w=nw, in_eps=eps)
        core = b.core.view(-1)[:T * cfg.value_dim].view(T, cfg.value_dim)
        self._row_parallel(self.lin[p + "out_proj"], core, T)

    def _conv_layer(self, i: int, T: int) -> None:
        """Gated short-convolution mixer: in_proj (RMSNorm in its prologue) -> C * fir(B * x) -> out_proj + residual."""
        cfg, b, w = self.cfg, self.buf, self.w
        p = f"text.layers.{i}.conv."
        H = cfg.conv_channels                  # this rank's channel block; out_proj is row-parallel over it
        bcx = b.mixed.view(-1)[:T * 3 * H].view(T, 3 * H)
        self.lin[p + "in_proj"](b.x[:T], out=bcx, prologue=K.PRO_RMSNORM, norm_w=w[f"text.layers.{i}.input_layernorm"],
                                eps=cfg.rms_norm_eps)
        core = b.core.view(-1)[:T * H].view(T, H)
        K.short_conv(bcx, w[p + "weight"], self.ring[i], b.positions, core, T)
        self._row_parallel(self.lin[p + "out_proj"], core, T)

    def _attn_layer(self, i: int, T: int) -> None:
        cfg, b, w = self.cfg, self.buf, self.w
        p = f"text.layers.{i}.attn."
        x, nw, eps = b.x[:T], w[f"text.layers.{i}.input_layernorm"], cfg.rms_norm_eps
        grp = self._siblings((p + "qg", p + "k", p + "v"))
        if grp is not None:
            grp(x, (b.qg[:T], b.k[:T], b.v[:T]), prologue=K.PRO_RMSNORM, norm_w=nw, eps=eps)
        else:
            side = self._fork()
            self.lin[p + "qg"](x, out=b.qg[:T], prologue=K.PRO_RMSNORM, norm_w=nw, eps=eps)
            with torch.cuda.stream(side) if side is not None else _NullCtx():
                self.lin[p + "k"](x, out=b.k[:T], prologue=K.PRO_RMSNORM, norm_w=nw, eps=eps)
                self.lin[p + "v"](x, out=b.v[:T], prologue=K.PRO_RMSNORM, norm_w=nw, eps=eps)
            self._join(side)
        self._attn_write(i, b.qg, b.k, b.v, b.positions, b.q, T)
        core = b.core.view(-1)[:T * cfg.q_dim].view(T, cfg.q_dim)
        self._attn_rows(i, T, core)
        self._row_parallel(self.lin[p + "o"], core, T, post_norm=w.get(f"text.layers.{i}.post_attn_out_norm"))

    def _mlp(self, i: int, T: int) -> None:
        cfg, b, w = self.cfg, self.buf, self.w
        if cfg.layer_is_moe(i):
            K.rmsnorm(b.x[:T], w[f"text.layers.{i}.post_attention_layernorm"], cfg.rms_norm_eps, out=b.h[:T])
            if self.comm is not None and hasattr(self.comm, "moe_forward"):
                self.comm.moe_forward(self.moe[i], b.h[:T], b.x[:T], T)
            elif self.comm is not None and self.comm.world > 1 and cfg.has_conv_layers:
                # tensor-parallel experts (the short-conv family: every rank holds a slice of every expert's inner width;
                # the hybrid MoE family keeps whole experts per rank and needs no sum): the routed sum is a
                # partial product, summed over the ranks before it joins the residual stream
                part = b.core.view(-1)[:T * cfg.hidden_size].view(T, cfg.hidden_size)
                self.moe[i].forward(b.h[:T], part, T, residual=False)
                self.comm.all_reduce_rows(part)
                K.residual_add(b.x[:T], part)
            else:
                self.moe[i].forward(b.h[:T], b.x[:T], T)
            return
        p = f"text.layers.{i}.mlp."
        self.lin[p + "gate_up"](b.x[:T], out=b.gate_up[:T], prologue=K.PRO_RMSNORM,
                                norm_w=w[f"text.layers.{i}.post_attention_layernorm"], eps=cfg.rms_norm_eps)
        self._row_parallel(self.lin[p + "down"], b.gate_up[:T], T,
                           prologue=K.PRO_GELU_MUL if cfg.mlp_act == "gelu_tanh" else K.PRO_SILU_MUL,
                           post_norm=w.get(f"text.layers.{i}.post_mlp_out_norm"))

    def _row_parallel(self, lin: Linear, x: torch.Tensor, T: int, prologue: int = 0, post_norm=None) -> None:
        """Row-parallel linear whose result is added to the residual stream ``buf.x``.  With ``post_norm`` (sandwich-norm
        families) the summed output is normalised first, so the add cannot ride in the product's epilogue."""
        b = self.buf
        if post_norm is not None:
            tmp = b.h[:T]                     # free here: the norms of a decode step live in the products' prologues
            if self.comm is None or self.comm.world == 1:
                lin(x, out=tmp, prologue=prologue)
            else:
                tmp.zero_()
                self.comm.row_parallel_linear(lin, x, tmp, prologue)
            K.norm_add(b.x[:T], tmp, post_norm, self.cfg.rms_norm_eps)
            return
        if self.comm is None or self.comm.world == 1:
            lin(x, out=b.x[:T], residual=b.x[:T], prologue=prologue)
        else:
            self.comm.row_parallel_linear(lin, x, b.x[:T], prologue)

    # race detector for tensor-parallel runs (R4DXB_TP_LOCKSTEP=1): before every forward call the ranks compare a fingerprint
    # of the call (kind, rows, position, checksum of the staged token ids) on the host and stop at the first difference,
    # instead of meeting later inside a collective with different shapes
    lockstep_checks = os.environ.get("R4DXB_TP_LOCKSTEP", "0") == "1"

    def _lockstep(self, kind: int, T: int, ids: torch.Tensor) -> None:
        if self.lockstep_checks and self.comm is not None and getattr(self.comm, "world", 1) > 1 and hasattr(self.comm, "check_lockstep"):
            self.comm.check_lockstep(kind, T, int(self.pos), int(ids[:T].to(torch.int64).sum().item()))

    # debug probe: ``probe(layer, residual_rows)`` is called after every layer of an eager call (never inside a captured
    # graph) - per-layer digests for locating where two runs diverge (utils/probe.py)
    probe = None

    def state_digest(self) -> Dict[str, float]:
        """Position and fp64 checksums of every piece of per-sequence state (recurrent states, conv rings, written KV
        blocks).  Equal digests mean equal state: tests compare them across a checkpoint round trip, a debugging session
        compares them between two runs or two ranks."""
        self.commit_pending()
        d: Dict[str, float] = {"pos": float(self.pos)}
        blocks = (self.pos + KV_BLOCK - 1) // KV_BLOCK
        for i, t in self.gdn_state.items():
            d[f"gdn.{i}"] = float(t.double().sum())
            d[f"ring.{i}"] = float(self.ring[i].double().sum())
        if blocks and self.kv_cache == "int4":         # what the written rows stand for
            rows = torch.arange(self.pos, dtype=torch.int32, device=self.device)
            for i, kv in self.kv.items():
                d[f"kv.{i}"] = float(sum(x.double().sum() for x in K.kv4_read(kv, self.block_table, rows)))
        elif blocks:
            tab = self.block_table[:blocks].long()
            live = (torch.arange(blocks * KV_BLOCK, device=self.device) < self.pos).view(blocks, 1, 1, KV_BLOCK, 1)
            for i, kv in self.kv.items():          # only rows below the position count: later rows of the last block are stale
                d[f"kv.{i}"] = float((kv[tab].view(torch.uint8).double() * live).sum())
        return d

    _key_limit = None      # per-row key limits of the chunk being prefilled (image blocks on sliding-window layers)

    # ---- residual rotation: rows enter the stack through Q and leave it through Q^T -------------------
    def _enter_stack(self, x: torch.Tensor) -> None:
        if self.rot is not None and self.layer_begin == 0:
            K.rotate_residual(x, self.rot[0], self.rot[1], inverse=False)

    def _leave_stack(self, x: torch.Tensor) -> None:
        if self.rot is not None and self.layer_end == self.cfg.num_hidden_layers:
            K.rotate_residual(x, self.rot[0], self.rot[1], inverse=True)

    # ---- forward --------------------------------------------------------------------------------
    def forward_rows(self, T: int, want_logits: bool = True, skip_embed: bool = False) -> None:
        """Runs the T rows staged in ``buf.ids`` / ``buf.positions``; results in ``buf.logits`` / ``buf.next_ids``.
        With ``skip_embed`` the caller has already placed the layer-0 input in ``buf.x``."""
        cfg, b, w = self.cfg, self.buf, self.w
        if not skip_embed:
            self._lockstep(0, T, b.ids)
        if not skip_embed and self.layer_begin == 0:
            K.embed_gather(b.ids[:T], w["text.embed_tokens"], out=b.x[:T])
            self._enter_stack(b.x[:T])
        for i in range(self.layer_begin, self.layer_end):
            if i in self.capture_layers:
                self._capture_rows(i, b.x[:T], T)
            # the two RMSNorms and the SwiGLU of a layer run inside the prologues of the linears
            if cfg.is_attention_layer(i):
                self._attn_layer(i, T)
            elif cfg.is_conv_layer(i):
                self._conv_layer(i, T)
            else:
                self._gdn_layer(i, T)
            self._mlp(i, T)
            if self.probe is not None and not torch.cuda.is_current_stream_capturing():
                self.probe(i, b.x[:T])
        self._leave_stack(b.x[:T])
        if want_logits and self.layer_end == cfg.num_hidden_layers:
            K.rmsnorm(b.x[:T], w["text.final_norm"], cfg.rms_norm_eps, out=b.h[:T])
            self.lin["lm_head"](b.h[:T], out=b.logits[:T])
            self._pick(T)

    def _pick(self, T: int) -> None:
        """``buf.next_ids[:T]`` out of the logits rows, with the status word of the products behind them in front."""
        b = self.buf
        K.argmax_rows(b.logits[:T], self.cfg.vocab_shard_begin, b.next_ids[:T], b.next_vals[:T], b.argmax_scratch, b.status_and_ids[:1])
        if self.comm is not None and self.comm.world > 1:
            self.comm.merge_argmax(b.next_ids[:T], b.next_vals[:T])

    # ---- feature capture for drafters that condition on intermediate residuals ----------------------
    capture_layers: tuple = ()

    def enable_capture(self, layers, max_rows: int) -> None:
        """Keeps the residual stream entering each of ``layers`` for the rows of the latest call in
        ``self.captured[j, :T]`` (reference: docs/dflash2.md:58 names the target layers a drafter reads)."""
        self.capture_layers = tuple(layers)
        self.captured = torch.zeros(len(self.capture_layers), max_rows, self.cfg.hidden_size, dtype=BF, device=self.device)

    def _capture_rows(self, layer: int, x: torch.Tensor, T: int) -> None:
        if T > self.captured.shape[1]:
            self.captured = torch.zeros(len(self.capture_layers), T, self.cfg.hidden_size, dtype=BF, device=self.device)
        dst = self.captured[self.capture_layers.index(layer), :T]
        dst.copy_(x)
        if self.rot is not None:              # consumers (drafters) read rows in the un-rotated basis
            K.rotate_residual(dst, self.rot[0], self.rot[1], inverse=True)

    def _stage(self, ids: torch.Tensor, pos0: int) -> int:
        T = ids.numel()
        b = self.buf
        b.ids[:T].copy_(ids.to(device=self.device, dtype=torch.int32), non_blocking=True)
        b.positions[:T].copy_(torch.arange(pos0, pos0 + T, dtype=torch.int32, device=self.device))
        return T

    def feed(self, ids: torch.Tensor, want_logits: bool = True, accepted: Optional[int] = None) -> None:
        """Feeds up to MAX_ROWS rows at the current position and commits all of them (or ``accepted``)."""
        T = self._stage(ids, self.pos)
        if self.pos + T > self.max_ctx:
            raise ValueError("context overflow")
        self.buf.n_replay.fill_(self.pending_rows)
        self.forward_rows(T, want_logits)
        n = T if accepted is None else accepted
        self.pending_rows = n
        self.pos += n

    def check_healthy(self, rows: int = 1) -> None:
        """Raises if a bounded device wait ran out since the last check: a timed-out collective leaves an un-reduced partial
        in the residual stream and a timed-out product NaN, from which a plausible first token id is picked, so a token read after it
        must not be trusted (one small device-to-host read per call).  ``rows`` (the row count of the call being checked) makes no
        difference: products of every row count have kernels whose waits report through the GEMM status word."""
        if self.comm is not None and self.comm.world > 1:
            self.comm.check_healthy()
        K.check_gemm_status(self.device)

    def _read_token(self, idx: int) -> int:
        self.last_row = idx              # the logits row this token was picked from (samplers read it)
        if idx == 0:                     # (a step's token: word and id as one number, 3 us less on the host than a list of two)
            pair = self.buf.status_and_ids[:2].view(torch.int64).item()
            status, tok = pair & 0xFFFFFFFF, pair >> 32
        else:
            status, *_, tok = self.buf.status_and_ids[:idx + 2].tolist()
        if self.comm is not None and self.comm.world > 1:
            self.comm.check_healthy()
        K.check_gemm_status(self.device, status)
        return tok

    def prefill_small(self, ids: torch.Tensor) -> int:
        """Feeds a prompt through the small-batch path (MAX_ROWS rows per call); returns the greedy next token."""
        ids = ids.to(torch.int32)
        n = ids.numel()
        s = 0
        while s < n:
            e = min(n, s + MAX_ROWS)
            self.feed(ids[s:e], want_logits=(e == n))
            s = e
        last = (n - 1) % MAX_ROWS
        return self._read_token(last)

    # ---- chunked prefill (tcgen05 GEMMs, long-chunk GDN scan, tensor-core attention) ----------------
    def _chunk_buffers(self, C: int) -> dict:
        cb = getattr(self, "_cb", None)
        if cb is not None and cb["C"] >= C:
            return cb
        cfg, dev = self.cfg, self.device
        H = cfg.hidden_size
        Hv, Hk, Dg = cfg.linear_num_value_heads, cfg.linear_num_key_heads, cfg.linear_key_head_dim
        kmax = max(H, cfg.value_dim, cfg.q_dim, cfg.intermediate_size)
        conv_w = 3 * H if cfg.has_conv_layers else 0
        e = lambda *s, dtype=BF: torch.empty(*s, dtype=dtype, device=dev)
        f32 = torch.float32
        # under tensor parallelism the residual stream of a chunk may live in peer-mapped memory (owners push rows into it)
        x_buf = self.comm.alloc_chunk_x(C, H) if hasattr(self.comm, "alloc_chunk_x") else e(C, H)
        cb = dict(C=C, ids=e(C, dtype=torch.int32), positions=e(C, dtype=torch.int32), x=x_buf, h=e(C, H),
                  xh=e(C * kmax, dtype=torch.float16), mixed=e(C * max(cfg.conv_dim, conv_w)), z=e(C, cfg.value_dim),
                  ab=e(C, 2 * Hv, dtype=f32), core=e(C * max(cfg.value_dim, cfg.q_dim, conv_w // 3)), qg=e(C, cfg.q_proj_dim),
                  k=e(C, cfg.kv_dim), v=e(C, cfg.kv_dim), q=e(C, cfg.q_dim), gate_up=e(C, 2 * cfg.intermediate_size),
                  gdn=dict(q=e(C, Hk, Dg, dtype=f32), k=e(C, Hk, Dg, dtype=f32), v=e(C, Hv, Dg, dtype=f32),
                           o=e(C, Hv, Dg, dtype=f32), eg=e(C, Hv, dtype=f32), beta=e(C, Hv, dtype=f32)))
        if Dg == 128 and Hv > 0 and C >= 128:
            cb["gdn"]["ws"] = e(K.gdn_chunk_ws_floats(C, Hv), dtype=f32)
        self._cb = cb
        return cb

    def commit_pending(self) -> None:
        """Folds the rows still sitting in the GDN logs into the base states (needed before a chunk scan)."""
        if self.pending_rows == 0:
            return
        cfg, b, w = self.cfg, self.buf, self.w
        b.n_replay.fill_(self.pending_rows)
        for i in self.gdn_state:
            p = f"text.layers.{i}.gdn."
            K.gdn_decode(b.mixed, b.z, b.ab, w[p + "conv1d_weight"], w[p + "A_log"], w[p + "dt_bias"], w[p + "norm_weight"],
                         self.ring[i], self.gdn_state[i], self.log_u[i], self.log_k[i], self.log_eg[i], b.positions,
                         b.n_replay, b.core, 0, cfg.linear_num_value_heads, cfg.linear_num_key_heads,
                         cfg.linear_key_head_dim, cfg.rms_norm_eps)
        self.pending_rows = 0
        b.n_replay.zero_()

    def forward_chunk(self, T: int, want_logits: bool, skip_embed: bool = False) -> None:
        """Runs T (> MAX_ROWS) rows staged in the chunk buffers at positions self.pos .. ; commits them."""
        cfg, w, cb = self.cfg, self.w, self._cb
        H = cfg.hidden_size
        Hv, Hk, Dg = cfg.linear_num_value_heads, cfg.linear_num_key_heads, cfg.linear_key_head_dim
        x, h = cb["x"][:T], cb["h"][:T]
        pos0 = self.pos
        self._lockstep(1, T, cb["ids"])
        if not skip_embed and self.layer_begin == 0:
            K.embed_gather(cb["ids"][:T], w["text.embed_tokens"], out=x)
            self._enter_stack(x)
        for i in range(self.layer_begin, self.layer_end):
            p = f"text.layers.{i}."
            if i in self.capture_layers:
                self._capture_rows(i, x, T)
            K.rmsnorm(x, w[p + "input_layernorm"], cfg.rms_norm_eps, out=h)
            if cfg.is_attention_layer(i):
                pa = p + "attn."
                qg, kk, vv, q = cb["qg"][:T], cb["k"][:T], cb["v"][:T], cb["q"][:T]
                self.lin[pa + "qg"].chunk(h, cb["xh"], qg)
                self.lin[pa + "k"].chunk(h, cb["xh"], kk)
                self.lin[pa + "v"].chunk(h, cb["xh"], vv)
                self._attn_write(i, qg, kk, vv, cb["positions"], q, T)
                core = cb["core"][:T * cfg.q_dim].view(T, cfg.q_dim)
                self._attn_chunk(i, q, qg, core, T, pos0)
                self._row_parallel_chunk(self.lin[pa + "o"], core, x, cb, post_norm=w.get(p + "post_attn_out_norm"))
            elif cfg.is_conv_layer(i):
                pc = p + "conv."
                Hc = cfg.conv_channels
                bcx = cb["mixed"][:T * 3 * Hc].view(T, 3 * Hc)
                self.lin[pc + "in_proj"].chunk(h, cb["xh"], bcx)
                core = cb["core"][:T * Hc].view(T, Hc)
                K.short_conv(bcx, w[pc + "weight"], self.ring[i], cb["positions"], core, T)
                self._row_parallel_chunk(self.lin[pc + "out_proj"], core, x, cb)
            else:
                pg = p + "gdn."
                mixed, z, ab = cb["mixed"][:T * cfg.conv_dim].view(T, cfg.conv_dim), cb["z"][:T], cb["ab"][:T]
                self.lin[pg + "in_proj_qkv"].chunk(h, cb["xh"], mixed)
                self.lin[pg + "in_proj_z"].chunk(h, cb["xh"], z)
                if self.ab_w[i].shape[0] % 4 == 0:
                    K.linear_tc(self.ab_w[i], h, out=ab)           # [T, 2 Hv] fp32 on the tensor cores (133 -> ~10 us per chunk)
                else:
                    K.bf16_gemv(self.ab_w[i], h, out=ab)
                core = cb["core"][:T * cfg.value_dim].view(T, cfg.value_dim)
                K.gdn_prefill(mixed, z, ab, w[pg + "conv1d_weight"], w[pg + "A_log"], w[pg + "dt_bias"],
                              w[pg + "norm_weight"], self.ring[i], self.gdn_state[i], cb["gdn"], core, T, Hv, Hk, Dg,
                              pos0, cfg.rms_norm_eps)
                self._row_parallel_chunk(self.lin[pg + "out_proj"], core, x, cb)
            K.rmsnorm(x, w[p + "post_attention_layernorm"], cfg.rms_norm_eps, out=h)
            if cfg.layer_is_moe(i):
                self._moe_chunk(i, h, x, T)
                continue
            pm = p + "mlp."
            gu = cb["gate_up"][:T]
            self.lin[pm + "gate_up"].chunk(h, cb["xh"], gu)
            self._row_parallel_chunk(self.lin[pm + "down"], gu, x, cb, fused_silu_mul=True, gelu=(cfg.mlp_act == "gelu_tanh"),
                                     post_norm=w.get(p + "post_mlp_out_norm"))
        self._leave_stack(x)
        if want_logits and self.layer_end == cfg.num_hidden_layers:
            b = self.buf
            K.rmsnorm(x[T - 1:T], w["text.final_norm"], cfg.rms_norm_eps, out=b.h[:1])
            self.lin["lm_head"](b.h[:1], out=b.logits[:1])
            self._pick(1)
        self.pos += T
        self.pending_rows = 0

    def _moe_chunk(self, i: int, h: torch.Tensor, x: torch.Tensor, T: int) -> None:
        """MoE block over a prefill chunk.  One GPU: all T rows are routed and planned at once and every expert's rows go
        through the grouped weight-streaming kernel eight at a time (as many passes as the fullest expert needs).
        Expert parallel: the exchange buffers are sized for decode, so the chunk goes through them in decode-sized slices."""
        if self.comm is not None and hasattr(self.comm, "moe_forward"):
            R = self.comm.R
            for s in range(0, T, R):
                e = min(T, s + R)
                self.comm.moe_forward(self.moe[i], h[s:e], x[s:e], e - s)
            return
        tp = self.comm is not None and self.comm.world > 1 and self.cfg.has_conv_layers      # experts sliced by inner width
        from .moe import MoeBlock
        blk = self._moe_chunk_blocks.get(i) if hasattr(self, "_moe_chunk_blocks") else None
        if blk is None or blk.logits.shape[0] < T:
            if not hasattr(self, "_moe_chunk_blocks"):
                self._moe_chunk_blocks = {}
            # one set of chunk-sized scratch buffers serves every layer; the expert stacks are the decode block's
            first = next(iter(self._moe_chunk_blocks.values()), None)
            if first is not None and first.logits.shape[0] >= T:
                blk = MoeBlock.__new__(MoeBlock)
                blk.__dict__.update(first.__dict__)
                src = self.moe[i]
                for name in ("gate_up", "down", "router", "shared_gate", "shared_gu", "shared_down", "expert_bias", "e_begin", "e_count", "ks_gu", "ks_dn",
                             "ks_gu_few", "ks_dn_few"):
                    setattr(blk, name, getattr(src, name))
            else:
                blk = MoeBlock(self.cfg, self.w, i, self.device, self._cb["C"], self.moe[i].e_begin, self.moe[i].e_count,
                               share_from=self.moe[i])
            self._moe_chunk_blocks[i] = blk
        if tp:
            part = self._cb["core"][:T * self.cfg.hidden_size].view(T, self.cfg.hidden_size)
            blk.forward(h, part, T, exact_rows=True, residual=False)
            self.comm.all_reduce_rows(part)
            K.residual_add(x, part)
        else:
            blk.forward(h, x, T, exact_rows=True)

    def _row_parallel_chunk(self, lin: Linear, inp: torch.Tensor, x: torch.Tensor, cb: dict,
                            fused_silu_mul: bool = False, gelu: bool = False, post_norm=None) -> None:
        if post_norm is not None or gelu:
            # sandwich-norm / GeGLU families: the fused tensor-parallel epilogues add into x directly, which a norm between
            # the product and the add rules out, so under tensor parallelism the bare product is summed over the ranks first
            tp = self.comm is not None and self.comm.world > 1
            if tp and os.environ.get("R4DXB_UNVALIDATED_TP") != "1":
                raise NotImplementedError("tensor-parallel prefill of sandwich-norm / GeGLU models is written but not validated "
                                          "on GPUs yet (set R4DXB_UNVALIDATED_TP=1 to run it anyway)")
            if post_norm is None and not tp:
                lin.chunk(inp, cb["xh"], x, residual=x, fused_silu_mul=fused_silu_mul, gelu=gelu)
                return
            tmp = cb["h"][:x.shape[0]]
            lin.chunk(inp, cb["xh"], tmp, fused_silu_mul=fused_silu_mul, gelu=gelu)
            if tp:
                self.comm.all_reduce_rows(tmp)
            if post_norm is None:
                K.residual_add(x, tmp)
            else:
                K.norm_add(x, tmp, post_norm, self.cfg.rms_norm_eps)
            return
        if self.comm is None or self.comm.world == 1:
            lin.chunk(inp, cb["xh"], x, residual=x, fused_silu_mul=fused_silu_mul)
        else:
            self.comm.row_parallel_chunk(lin, inp, x, cb, fused_silu_mul)

    def reserve_prefill(self, rows: int) -> None:
        """Allocates the chunk workspaces for prefill chunks of up to ``rows`` rows ahead of time."""
        self._chunk_buffers(rows)

    @staticmethod
    def auto_chunk(n: int) -> int:
        """Rows per prefill chunk: the whole prompt up to 8192 rows, 8192-row chunks beyond.  Measured on 16 layers of the
        27B geometry with an 8192-token prompt: 1536 / 4096 / 8192-row chunks take 162.8 / 154.5 / 148.8 ms on one GPU and
        58.0 / 39.9 / 36.3 ms at the shard shapes of 8 ranks (whose products are an eighth as wide: only long chunks give
        them enough token tiles to fill the 148 SMs); 32k tokens: 650 ms with 8192-row chunks against 679 ms with 4096."""
        return 8192

    def prefill(self, ids: torch.Tensor, chunk: Optional[int] = None, hook=None, embed_overrides=None, image_blocks=None) -> int:
        """Cold or warm prefill of ``ids`` at the current position; returns the greedy next token.
        ``hook(start, T, hidden_rows)`` is called after every chunk with the final hidden states of its rows
        (drafters keep their own caches in lock-step with it).  ``image_blocks``: [start, end) runs of image rows
        (indices into ``ids``) that attend to each other in both directions on sliding-window layers; chunks never
        cut such a block."""
        ids = ids.to(torch.int32)
        n = ids.numel()
        chunk = chunk or self.auto_chunk(n)
        if embed_overrides is not None or image_blocks:
            return self._prefill_with_embeds(ids, chunk, hook, embed_overrides, image_blocks)
        if n <= MAX_ROWS:
            tok = self.prefill_small(ids)
            if hook is not None:
                hook(0, n, self.buf.x[:n])
            return tok
        if self.pos + n > self.max_ctx:
            raise ValueError("context overflow")
        self.commit_pending()
        cb = self._chunk_buffers(min(chunk, n))
        step = min(chunk, cb["C"])         # the buffers may be larger (kept from an earlier call): the chunk size is what was asked for
        s = 0
        last_small = False
        while s < n:
            e = min(n, s + step)
            T = e - s
            if T <= MAX_ROWS:
                # short tail: the small-batch path logs its rows instead of committing them
                self.feed(ids[s:e], want_logits=True)
                last_small = True
                if hook is not None:
                    hook(s, T, self.buf.x[:T])
            else:
                cb["ids"][:T].copy_(ids[s:e].to(self.device), non_blocking=True)
                cb["positions"][:T].copy_(torch.arange(self.pos, self.pos + T, dtype=torch.int32, device=self.device))
                self.forward_chunk(T, want_logits=(e == n))
                if hook is not None:
                    hook(s, T, cb["x"][:T])
            s = e
        K.check_gemm_status(self.device)
        if last_small:
            return self._read_token((n - 1) % step)
        return self._read_token(0)

    def _prefill_with_embeds(self, ids: torch.Tensor, chunk: int, hook, overrides, image_blocks=None) -> int:
        """Prefill in which some rows' input embeddings come from outside (image tokens): ``overrides`` =
        (positions int64 [M] relative to ``ids``, rows bf16 [M, H]).  Always runs the chunk path
        (reference: src/model/model.cpp:2062-2113 injects vision embeddings the same way).  With ``image_blocks`` the
        chunks are planned so that no block is cut, and the sliding-window layers get a per-row key limit: a row of a block
        sees its whole block (reference: src/vision/gemma_vision.cpp plans chunks and masks the same way)."""
        n = ids.numel()
        if overrides is not None:
            pos, rows = overrides
            pos = pos.to(self.device, torch.long)
            rows = rows.to(self.device, BF)
        else:
            pos, rows = torch.zeros(0, dtype=torch.long, device=self.device), None
        if self.pos + n > self.max_ctx:
            raise ValueError("context overflow")
        self.commit_pending()
        blocks = [(int(a), int(b)) for a, b in (image_blocks or [])]
        if blocks:
            from .gemma_vision import key_limit_ext, plan_prefill_chunks
            plan = plan_prefill_chunks(n, blocks, max(MAX_ROWS + 1, min(chunk, n)))
            base = self.pos
        else:
            plan = None
        cb = self._chunk_buffers(max([MAX_ROWS + 1, min(chunk, n)] + ([t for _, t in plan] if plan else [])))
        s = 0
        ci = 0
        while s < n:
            e = min(n, s + cb["C"]) if plan is None else s + plan[ci][1]
            ci += 1
            T = e - s
            if blocks:
                lim = key_limit_ext(s, T, blocks)
                lim = torch.where(lim >= 0, lim + base, lim)         # absolute key positions
                self._key_limit = lim.to(self.device) if bool((lim >= 0).any()) else None
            cb["ids"][:T].copy_(ids[s:e].to(self.device), non_blocking=True)
            cb["positions"][:T].copy_(torch.arange(self.pos, self.pos + T, dtype=torch.int32, device=self.device))
            x = cb["x"][:T]
            K.embed_gather(cb["ids"][:T], self.w["text.embed_tokens"], out=x)
            sel = (pos >= s) & (pos < e)
            if bool(sel.any()):
                x[pos[sel] - s] = rows[sel]
            self._enter_stack(x)                 # spliced rows are rotated along with the text rows
            try:
                self.forward_chunk(T, want_logits=(e == n), skip_embed=True)
            finally:
                self._key_limit = None
            if hook is not None:
                hook(s, T, x)
            s = e
        K.check_gemm_status(self.device)
        return self._read_token(0)

    def logits_rows(self, T: int) -> torch.Tensor:
        return self.buf.logits[:T]

    # ---- speculative window -----------------------------------------------------------------------
    def verify_window(self, anchor: int, drafts: List[int]) -> List[int]:
        """Feeds [anchor, d1..dm] (m <= MAX_ROWS - 1), accepts the longest prefix of drafts the target agrees
        with (greedy, lossless) and commits exactly those rows.  Returns the emitted tokens: accepted drafts
        plus one correction / bonus token (reference: src/model/model.cpp:2694-2975, 3344-3426)."""
        m = len(drafts)
        if m + 1 > MAX_ROWS:
            raise ValueError("speculative window too long")
        ids = torch.tensor([anchor] + list(drafts), dtype=torch.int32)
        T = self._stage(ids, self.pos)
        if self.pos + T > self.max_ctx:
            raise ValueError("context overflow")
        b = self.buf
        b.n_replay.fill_(self.pending_rows)
        self._run_rows(T)
        if not hasattr(self, "_spec_out"):
            self._spec_out = torch.zeros(MAX_ROWS + 2, dtype=torch.int32, device=self.device)
        K.spec_accept(b.next_ids, b.ids[1:], T, self._spec_out, None)
        res = self._spec_out[:T + 1].tolist()        # one small read-back per round
        self.check_healthy(T)
        n = res[0]
        self.pending_rows = n
        self.pos += n
        return res[1:1 + n]

    def _run_rows(self, T: int) -> None:
        """The staged T rows through the layer stack and the head: a replay of the captured graph for this row count when
        there is one (``enable_graphs((T,))``: a window is ~360 launches, which an eager call issues one by one), else
        eagerly.  The graph's trailing bookkeeping only touches buffers every caller of this method stages again."""
        g = self._graphs.get(T)
        if g is not None:
            g.replay()
        else:
            self.forward_rows(T, True)

    def window_logits(self, anchor: int, drafts: List[int]) -> torch.Tensor:
        """Runs the window [anchor, d1..dm] and returns its fp32 logits rows WITHOUT committing anything; follow with
        ``commit_window(n)`` (sampled speculation resolves acceptance on the host, one draw per row)."""
        m = len(drafts)
        if m + 1 > MAX_ROWS:
            raise ValueError("speculative window too long")
        ids = torch.tensor([anchor] + list(drafts), dtype=torch.int32)
        T = self._stage(ids, self.pos)
        if self.pos + T > self.max_ctx:
            raise ValueError("context overflow")
        self.buf.n_replay.fill_(self.pending_rows)
        self._run_rows(T)
        self.check_healthy(T)
        self._window_rows = T
        return self.buf.logits[:T]

    def commit_window(self, n: int) -> None:
        if not 1 <= n <= getattr(self, "_window_rows", 0):
            raise ValueError("commit_window outside the last window")
        self.pending_rows = n
        self.pos += n
        self._window_rows = 0

    # ---- prompt checkpoint ---------------------------------------------------------------------------
    def save_checkpoint(self) -> dict:
        """Snapshot of the recurrent state (KV needs no copy: it is overwritten by position)
        (reference: src/model/model.h:361-379)."""
        self.commit_pending()
        return {"pos": self.pos, "gdn": {i: t.clone() for i, t in self.gdn_state.items()},
                "ring": {i: t.clone() for i, t in self.ring.items()}}

    def restore_checkpoint(self, ck: dict) -> None:
        for i, t in ck["gdn"].items():
            self.gdn_state[i].copy_(t)
        for i, t in ck["ring"].items():
            self.ring[i].copy_(t)
        self.pos = ck["pos"]
        self.pending_rows = 0
        self.buf.n_replay.zero_()

    def decode_step_logits(self, token: int) -> torch.Tensor:
        """Eager single step returning this rank's fp32 logits row (sampling path)."""
        self.feed(torch.tensor([token], dtype=torch.int32))
        self.check_healthy()
        return self.buf.logits[0]

    # ---- graph decode ---------------------------------------------------------------------------
    def _capture(self, T: int) -> torch.cuda.CUDAGraph:
        b = self.buf
        # warm-up on a side stream (sets kernel attributes, loads modules) without touching live state
        snap = self._snapshot()
        # warm-up rows live in the spare KV block past max_ctx, so no real cache row is touched
        b.positions.copy_(torch.arange(self.max_ctx, self.max_ctx + MAX_ROWS, dtype=torch.int32, device=self.device))
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            self._graph_body(T)
        torch.cuda.current_stream().wait_stream(s)
        self._restore(snap)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            self._graph_body(T)
        self._restore(snap)
        return g

    def _graph_body(self, T: int) -> None:
        b = self.buf
        self.forward_rows(T, True)
        # device-side bookkeeping so the graph can be replayed back to back
        b.ids[:1].copy_(b.next_ids[T - 1:T])
        b.positions.add_(T)
        b.n_replay.fill_(T)

    def _snapshot(self):
        b = self.buf
        snap = {"ids": b.ids.clone(), "pos": b.positions.clone(), "nr": b.n_replay.clone(), "x": b.x.clone()}
        snap["kvrow"] = {}
        snap["gdn"] = {i: t.clone() for i, t in self.gdn_state.items()}
        snap["ring"] = {i: t.clone() for i, t in self.ring.items()}
        snap["log"] = {i: (self.log_u[i].clone(), self.log_k[i].clone(), self.log_eg[i].clone()) for i in self.log_u}
        return snap

    def _restore(self, snap) -> None:
        b = self.buf
        b.ids.copy_(snap["ids"]); b.positions.copy_(snap["pos"]); b.n_replay.copy_(snap["nr"]); b.x.copy_(snap["x"])
        for i, t in snap["gdn"].items():
            self.gdn_state[i].copy_(t)
        for i, t in snap["ring"].items():
            self.ring[i].copy_(t)
        for i, (u, k, eg) in snap["log"].items():
            self.log_u[i].copy_(u); self.log_k[i].copy_(k); self.log_eg[i].copy_(eg)

    def enable_graphs(self, rows=(1,)) -> None:
        for T in rows:
            if T not in self._graphs:
                self._graphs[T] = self._capture(T)

    def decode_begin(self, first_token: int) -> None:
        """Stages the token / position / commit count for graph replays starting at the current position."""
        b = self.buf
        b.ids[:1].fill_(first_token)
        b.positions.copy_(torch.arange(self.pos, self.pos + MAX_ROWS, dtype=torch.int32, device=self.device))
        b.n_replay.fill_(self.pending_rows)

    def decode_step_graph(self) -> None:
        """One greedy step: consumes ``buf.ids[0]``, leaves the next token in ``buf.ids[0]`` / ``buf.next_ids[0]``."""
        if self.pos + 1 > self.max_ctx:
            raise ValueError("context overflow")
        self._graphs[1].replay()
        self.pos += 1
        self.pending_rows = 1

    def decode_step_greedy(self, token: int) -> int:
        """Eager single step (no graph): feed one token, return the greedy next token."""
        self.feed(torch.tensor([token], dtype=torch.int32))
        return self._read_token(0)

    def generate_greedy(self, prompt: torch.Tensor, n: int, use_graph: bool = True) -> List[int]:
        tok = self.prefill(prompt)
        out = [tok]
        if n <= 1:
            return out
        if use_graph:
            self.enable_graphs((1,))
            self.decode_begin(tok)
            toks = torch.empty(n - 1, dtype=torch.int32, device=self.device)
            for j in range(n - 1):
                self.decode_step_graph()
                toks[j:j + 1].copy_(self.buf.next_ids[:1])
            out += toks.tolist()
            self.check_healthy()
        else:
            for _ in range(n - 1):
                tok = self.decode_step_greedy(tok)
                out.append(tok)
        return out
