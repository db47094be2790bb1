"""Tensor-parallel Llama-style decoder stack built on the fused GEMM + collective kernels.

Per layer, on every rank (W ranks, tokens T = batch x seq, hidden H, SwiGLU width I):

    x_shard [T/W, H]   (the residual stream is token-sharded between blocks)
      RMSNorm -> written straight into this rank's rows of the gathered activation matrix
      all-gather -> GEMM   qkv   = gather(xn) [T, H]   @ Wqkv_r^T [H, 3H/W]       (column-parallel, fused)
      (norms of query and key heads, rotation by position, keys and values into the cache: one kernel, where configured)
      causal attention over this rank's H/W / head_dim heads, or of the newest tokens over the cache
      GEMM -> all-reduce   o     = attn [T, H/W]       @ Wo_r^T   [H/W, H]        (row-parallel, fused)
      x_shard += o[own rows]
      RMSNorm -> gathered matrix; all-gather -> GEMM  gate|up = gather(xn) @ Wgu_r^T [H, 2I/W]
      SwiGLU; GEMM -> all-reduce  down = h [T, I/W] @ Wd_r^T [I/W, H];  x_shard += down[own rows]

The reference has no model code; its fused kernels are the ingredients (``docs/FINEGRAINED_OVERLAP.md:23-31``
describes the row-parallel and column-parallel splits).  ``TPDecoderBaseline`` is the same network with cuBLAS GEMMs
and NCCL ``all_gather_into_tensor`` / ``all_reduce``; ``reference_forward`` is the unsharded fp32 oracle.
The attention core of the fused stack is this repository's tcgen05 kernel (``iris_b200/ops/attention.py``) whenever
the head dimension is 128 and the sequence length a multiple of 128 (with positions, head norms or a cache: any length); the
baseline stack (and the fused one for other shapes, or with ``attention="sdpa"``) calls
``torch.nn.functional.scaled_dot_product_attention``.  Grouped heads and sliding windows (``attention_window_fwd``, any sequence
length), and single tokens over a cache (``paged_attention``), need the own kernels.

Serving: a decoder of whole prompts (``seq`` rows to a sequence) and one of single tokens (``seq=1``, ``weights=`` the first one's)
share a paged cache (``iris_b200/ops/paged.py``, :meth:`TPDecoder.make_cache`).  ``forward(x, cache=..., new_lens=...)`` takes the
pages of the new tokens, writes their keys and values and, with ``seq=1``, attends over the pages (``paged_attention``); nothing
waits for the GPU, so that a step can be captured and replayed.
"""
from __future__ import annotations

import os
from dataclasses import dataclass
from typing import List, Optional, Sequence, Union

import torch
import torch.nn.functional as F

from ..context import Iris
from ..ops import attention as A
from ..ops import elementwise as E
from ..ops import gemm as G
from ..ops import paged as P
from ..ops import rotary as R


@dataclass
class TPConfig:
    hidden: int = 4096
    n_heads: int = 32
    head_dim: int = 128
    intermediate: int = 11008
    eps: float = 1e-6
    n_layers: int = 4
    batch: int = 8
    seq: int = 2048
    seed: int = 4
    std: float = 0.02
    n_kv_heads: int = 0       # 0: as many as query heads
    qk_norm: bool = False     # norms of query and key heads (weights per component)
    rope_theta: float = 0.0   # 0: no rotation; else cosines and sines for `positions` positions
    rotary_dim: int = 0       # rotated part of a head; 0: all of it
    interleaved: bool = False
    positions: int = 0        # 0: `seq`
    window: int = 0           # 0: no window
    sinks: int = 0

    @property
    def tokens(self) -> int:
        return self.batch * self.seq

    @property
    def kv_heads(self) -> int:
        return self.n_kv_heads or self.n_heads

    @property
    def plain(self) -> bool:
        """Whether attention is over all keys, as many as query heads, without positions."""
        return self.kv_heads == self.n_heads and not (self.qk_norm or self.rope_theta or self.window)


def layer_weights(cfg: TPConfig, layer: int, device) -> dict:
    """Full (unsharded) bf16 weights of one layer, identical on every rank: N(0, std) from ``seed + layer``."""
    g = torch.Generator(device=device).manual_seed(cfg.seed * 1000 + layer)
    H, I = cfg.hidden, cfg.intermediate

    def w(rows, cols):
        return (torch.randn((rows, cols), generator=g, device=device) * cfg.std).to(torch.bfloat16)
    kv = cfg.kv_heads * cfg.head_dim
    full = {"wq": w(H, H), "wk": w(kv, H), "wv": w(kv, H), "wo": w(H, H), "wg": w(I, H), "wu": w(I, H), "wd": w(H, I),
            "norm1": torch.ones(H, device=device, dtype=torch.bfloat16),
            "norm2": torch.ones(H, device=device, dtype=torch.bfloat16)}
    for name in ("q_norm", "k_norm") if cfg.qk_norm else ():
        full[name] = (1 + 0.1 * torch.randn(cfg.head_dim, generator=g, device=device)).to(torch.bfloat16)
    return full


def shard_weights(full: dict, cfg: TPConfig, rank: int, world: int) -> dict:
    H, I = cfg.hidden, cfg.intermediate
    hs, is_ = H // world, I // world
    r0, r1 = rank * hs, (rank + 1) * hs
    ks = cfg.kv_heads * cfg.head_dim // world
    k0, k1 = rank * ks, (rank + 1) * ks
    i0, i1 = rank * is_, (rank + 1) * is_
    return {
        "wqkv": torch.cat([full["wq"][r0:r1], full["wk"][k0:k1], full["wv"][k0:k1]], 0).contiguous(),  # [3H/W, H]
        "wo": full["wo"][:, r0:r1].contiguous(),                                                     # [H, H/W]
        "wgu": torch.cat([full["wg"][i0:i1], full["wu"][i0:i1]], 0).contiguous(),                      # [2I/W, H]
        "wd": full["wd"][:, i0:i1].contiguous(),                                                     # [H, I/W]
        "norm1": full["norm1"], "norm2": full["norm2"], "q_norm": full.get("q_norm"), "k_norm": full.get("k_norm")}


def attention(qkv: torch.Tensor, cfg: TPConfig, heads_local: int, out: torch.Tensor) -> torch.Tensor:
    """Causal self-attention over the local heads.  qkv: [T, 3 * heads_local * d]; out: [T, heads_local * d]."""
    B, S, d = cfg.batch, cfg.seq, cfg.head_dim
    hl = heads_local * d
    q = qkv[:, :hl].view(B, S, heads_local, d).transpose(1, 2)
    k = qkv[:, hl:2 * hl].view(B, S, heads_local, d).transpose(1, 2)
    v = qkv[:, 2 * hl:].view(B, S, heads_local, d).transpose(1, 2)
    o = F.scaled_dot_product_attention(q, k, v, is_causal=True)
    out.view(B, S, heads_local, d).copy_(o.transpose(1, 2))
    return out


def attention_iris(qkv: torch.Tensor, cfg: TPConfig, heads_local: int, out: torch.Tensor, status=None) -> torch.Tensor:
    """The same on the tcgen05 kernel: reads Q, K, V straight out of the projection's output, writes ``out`` in place
    (no transposes, no copies)."""
    return A.attention_fwd(qkv, out, cfg.batch, cfg.seq, heads_local, causal=True, status=status)


class TPDecoder:
    """Fused implementation.  ``ctxs``: one ``Iris`` (one process per GPU) or all members of ``Iris.local_world``.
    ``variant``: how the row-parallel projections reduce (an all-reduce variant of ``gemm_all_reduce``, ``"auto"``, or
    ``"reduce_scatter"``); ``attention``: ``"iris"`` (own kernel, when the shape allows) or ``"sdpa"``; ``weights``: another
    decoder of the same ranks whose weights to use."""

    def __init__(self, ctxs: Union[Iris, Sequence[Iris]], cfg: TPConfig, variant: str = "two_shot", ag_slices: int = 8,
                 attention: str = "iris", weights: Optional["TPDecoder"] = None):
        self.ctxs: List[Iris] = [ctxs] if isinstance(ctxs, Iris) else list(ctxs)
        self.cfg = cfg
        c0 = self.ctxs[0]
        self.world = c0.get_num_ranks()
        self.ranks = [c.get_rank() for c in self.ctxs]
        dev = c0.device
        W, T, H, I = self.world, cfg.tokens, cfg.hidden, cfg.intermediate
        if cfg.n_heads % W or I % W or T % W or (I // W) % 8:
            raise ValueError("heads, intermediate size and tokens must divide by the number of ranks")
        if cfg.n_heads % cfg.kv_heads or cfg.kv_heads % W:
            raise ValueError("key heads must divide the query heads, and by the number of ranks")
        if cfg.hidden != cfg.n_heads * cfg.head_dim and not cfg.plain:
            raise ValueError("the hidden size must be that of all heads")
        if cfg.rope_theta and cfg.positions and cfg.positions < cfg.seq:
            raise ValueError("fewer positions than rows of a sequence")
        if weights is not None and (weights.ranks != self.ranks or len(weights.layers) != cfg.n_layers or any(
                getattr(weights.cfg, f) != getattr(cfg, f)
                for f in ("hidden", "n_heads", "head_dim", "intermediate", "kv_heads", "qk_norm"))):
            raise ValueError("weights of a decoder of other ranks or sizes")
        self.kv_heads_local = cfg.kv_heads // W
        self.windowed = cfg.window > 0 or cfg.kv_heads != cfg.n_heads
        if self.windowed and cfg.seq > 1 and (attention != "iris" or cfg.head_dim != A.HEAD_DIM):
            raise ValueError(f"windows and grouped heads need the own attention kernel (head dimension {A.HEAD_DIM})")
        # "reduce_scatter": the row-parallel projections deliver only this rank's token rows (all the layer uses)
        self.scatter = variant == "reduce_scatter"

        def row_parallel(a, bt):
            if self.scatter:
                return G.gemm_reduce_scatter(self.ctxs, a, bt)
            return G.gemm_all_reduce(self.ctxs, a, bt, variant=variant)

        def column_parallel(bt, **kw):
            """The product of the gathered rows, and the matrix to put one's own rows of them into."""
            if W == 1 and T % 128:   # (the all-gather prologue moves blocks of 128 rows, which alone has nothing to gather)
                a = torch.empty((T, H), dtype=torch.bfloat16, device=dev)
                return G.FusedGemm(self.ctxs, [a], bt, "store", **kw), [a]
            op = G.all_gather_gemm(self.ctxs, T, bt, ag_slices=ag_slices, **kw)
            return op, op.a_full
        self.heads_local = cfg.n_heads // W
        self.own_ragged = attention == "iris" and cfg.head_dim == A.HEAD_DIM      # any length, with positions, norms or a cache
        self.own_attention = self.own_ragged and cfg.seq % 128 == 0
        self.ts = T // W
        nl = len(self.ctxs)
        # one rank: the gate / up projection applies the SwiGLU on its way out (its own kernel otherwise)
        self.fused_swiglu = W == 1 and "IRIS_STREAM_K" not in os.environ
        ints = dict(dtype=torch.int32, device=dev)
        self.positions = torch.arange(cfg.seq, **ints).repeat(cfg.batch)                     # without a cache
        self.cache_positions, self.slots = torch.empty(T, **ints), torch.empty(T, **ints)    # of the last call with one
        self.rotation = None
        if cfg.rope_theta:
            self.rotation = R.rotary_table(cfg.positions or cfg.seq, cfg.rotary_dim or cfg.head_dim, cfg.rope_theta, device=dev)
        self.attn = [torch.empty((T, H // W), dtype=torch.bfloat16, device=dev) for _ in range(nl)]
        self.h = [torch.empty((T, I // W), dtype=torch.bfloat16, device=dev) for _ in range(nl)]
        self.layers = []
        for layer in range(cfg.n_layers):
            if weights is not None:
                sh = weights.layers[layer]["w"]
            else:
                full = layer_weights(cfg, layer, dev)
                sh = [shard_weights(full, cfg, r, W) for r in self.ranks]
                del full
            qkv, qkv_in = column_parallel([s["wqkv"] for s in sh])
            gu, gu_in = column_parallel([s["wgu"] for s in sh], **(dict(swiglu=True, out=self.h) if self.fused_swiglu else {}))
            ops = {
                "w": sh,
                "qkv": qkv, "qkv_in": qkv_in,
                "o": row_parallel(self.attn, [s["wo"] for s in sh]),
                "gu": gu, "gu_in": gu_in,
                "down": row_parallel(self.h, [s["wd"] for s in sh]),
            }
            self.layers.append(ops)
        self.kernel_launches = 0

    def rows(self, local: int) -> slice:
        r = self.ranks[local]
        return slice(r * self.ts, (r + 1) * self.ts)

    def make_cache(self, pages: int, page_size: int, max_batch: int, max_len: int) -> List[P.PagedCache]:
        """A paged cache for every local rank's key heads, one to each."""
        return [P.PagedCache(self.cfg.n_layers, pages, page_size, self.kv_heads_local, self.cfg.head_dim, max_batch, max_len,
                             device=c.device) for c in self.ctxs]

    def forward(self, x_shards: Sequence[torch.Tensor], timers=None, cache: Optional[Sequence[P.PagedCache]] = None,
                new_lens: Optional[torch.Tensor] = None) -> Sequence[torch.Tensor]:
        """``x_shards[l]``: [T/W, H] bf16 of local rank l; updated in place and returned.  ``timers``: optional
        callable ``timers(name)`` invoked before every phase (per-phase breakdowns with CUDA events).

        ``cache``: one paged cache per local rank (:meth:`make_cache`), of ``batch`` requests.  ``new_lens`` int32 [batch] says how
        many of each request's ``seq`` rows are tokens (the first ones); the cache takes pages for them and their keys and
        values.  With ``seq`` rows and more than one, these are whole prompts, which attend over their own rows alone, so that a
        request that holds tokens already gets nothing; with ``seq=1`` the newest token of each request attends over its pages
        (with peers, ``batch`` is a multiple of 128 per rank, as the rows of every fused all-gather -> GEMM).  Rows of no token,
        and of requests that got nothing (:func:`iris_b200.ops.paged.reserve_slots`; their length in the cache stays) may hold anything and give no meaningful output."""
        cfg, nl = self.cfg, len(self.ctxs)
        n = 0
        tick = timers if timers is not None else (lambda name: None)
        if (cache is None) != (new_lens is None):
            raise ValueError("cache and new_lens belong together")
        if cache is not None:
            if len(cache) != nl or any(c.data.shape[0] != cfg.n_layers or c.data.shape[4:] != (self.kv_heads_local, cfg.head_dim) or
                                       c.lens.shape[0] != cfg.batch or c.data.dtype != torch.bfloat16 for c in cache):
                raise ValueError("the cache does not fit this decoder (make_cache)")
            if self.rotation is not None and any(c.max_len > self.rotation.shape[0] for c in cache):
                raise ValueError("the cache holds more positions than there are angles for (TPConfig.positions)")
            if cfg.seq == 1 and cfg.head_dim not in P.HEAD_DIMS:
                raise ValueError(f"single tokens over a cache need heads of 64, 128 or 256, not {cfg.head_dim}")
            tick("reserve")
            for l in range(nl):
                cache[l].reserve(new_lens, self.slots, self.cache_positions, row_stride=cfg.seq, fresh=cfg.seq > 1)
            n += nl
            if cfg.seq > 1:
                # A prompt's padding may hold anything, and infinity or NaN would reach the tokens that share its tile of keys with
                # a weight of zero (single tokens share no tile): zeros stay finite through all layers.
                for l in range(nl):
                    x_shards[l].masked_fill_((self.cache_positions[self.rows(l)] < 0)[:, None], 0)
        pending = None   # output of the previous layer's down projection, not yet added to the residual stream
        for layer, ops in enumerate(self.layers):
            tick("norm")
            for l in range(nl):
                dst = ops["qkv_in"][l][self.rows(l)]
                if pending is None:
                    E.rmsnorm(x_shards[l], ops["w"][l]["norm1"], dst, cfg.eps)
                else:   # the previous layer's residual add rides along with this layer's first norm
                    E.add_rmsnorm(x_shards[l], pending[l], ops["w"][l]["norm1"], dst, cfg.eps)
            tick("qkv_ag_gemm")
            qkv = ops["qkv"]()
            tick("attention")
            for l in range(nl):
                if cache is not None or not cfg.plain:
                    self._attend(qkv[l], l, layer, cache)
                elif self.own_attention:
                    attention_iris(qkv[l], cfg, self.heads_local, self.attn[l], status=self.ctxs[l].status)
                else:
                    attention(qkv[l], cfg, self.heads_local, self.attn[l])
            tick("o_gemm_ar")
            o = ops["o"]()
            tick("norm")
            for l in range(nl):   # residual add and the next norm in one pass, written into the gathered matrix
                E.add_rmsnorm(x_shards[l], o[l] if self.scatter else o[l][self.rows(l)], ops["w"][l]["norm2"],
                              ops["gu_in"][l][self.rows(l)], cfg.eps)
            tick("gu_ag_gemm")
            gu = ops["gu"]()
            tick("swiglu")
            for l in range(nl if not self.fused_swiglu else 0):
                E.swiglu(gu[l], self.h[l])
            tick("down_gemm_ar")
            d = ops["down"]()
            pending = [d[l] if self.scatter else d[l][self.rows(l)] for l in range(nl)]
            n += nl if cache is not None or not cfg.plain else 0
            n += 4 + (3 if self.fused_swiglu else 4) * nl   # 4 fused GEMMs; per rank: norm, attention, add+norm, SwiGLU
        tick("norm")
        for l in range(nl):
            E.residual_add(x_shards[l], pending[l])
        n += nl
        tick("end")
        self.kernel_launches += n
        return x_shards

    def _attend(self, qkv: torch.Tensor, l: int, layer: int, cache) -> None:
        """Norms, rotation and cache, in place, then attention of the kind that the configuration and the cache ask for."""
        cfg, w, status = self.cfg, self.layers[layer]["w"][l], self.ctxs[l].status
        hl, kl, d = self.heads_local, self.kv_heads_local, cfg.head_dim
        decode = cache is not None and cfg.seq == 1
        if cache is not None or cfg.qk_norm or cfg.rope_theta:
            kept = {} if cache is None else dict(k_cache=cache[l].k(layer), v_cache=cache[l].v(layer), slots=self.slots)
            R.qk_norm_rope(qkv, qkv[:, :hl * d] if decode else qkv, self.positions if cache is None else self.cache_positions,
                           self.rotation, hl, kl, d, q_weight=w["q_norm"], k_weight=w["k_norm"], eps=cfg.eps,
                           interleaved=cfg.interleaved, status=status, **kept)
        if decode:
            q, out = (t[:, :hl * d].unflatten(1, (hl, d)) for t in (qkv, self.attn[l]))
            P.paged_attention(q, cache[l].k(layer), cache[l].v(layer), cache[l].block_table, cache[l].lens, out,
                              window=cfg.window, sinks=cfg.sinks, status=status)
        elif self.windowed or (self.own_ragged and cfg.seq % 128):
            A.attention_window_fwd(qkv, self.attn[l], cfg.batch, cfg.seq, hl, kl, window=cfg.window or cfg.seq, sinks=cfg.sinks,
                                   status=status)
        elif self.own_attention:
            attention_iris(qkv, cfg, hl, self.attn[l], status=status)
        else:
            attention(qkv, cfg, hl, self.attn[l])

    def capture(self, x_shards: Sequence[torch.Tensor], cache: Optional[Sequence[P.PagedCache]] = None,
                new_lens: Optional[torch.Tensor] = None) -> "torch.cuda.CUDAGraph":
        """Record one forward pass over ``x_shards`` (updated in place, as ``forward`` does) into a CUDA graph and
        return it; ``graph.replay()`` then runs the whole pass, all ranks' collectives included, with one submission
        instead of one launch per kernel.  Every rank captures and replays the same number of times.  The fused
        kernels keep their call numbers (flag targets, buffer parity) in device memory, so a recorded launch is
        valid for every replay and may be mixed with ordinary ``forward`` calls.  With a cache, every replay takes
        ``new_lens`` (its values at that time) further tokens."""
        torch.cuda.synchronize(self.ctxs[0].device)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            self.forward(x_shards, cache=cache, new_lens=new_lens)
        return graph

    def check(self) -> None:
        torch.cuda.synchronize(self.ctxs[0].device)
        for c in self.ctxs:
            c.check_status()

    def close(self) -> None:
        for ops in self.layers:
            for k in ("qkv", "o", "gu", "down"):
                ops[k].close()


class TPDecoderBaseline:
    """Same network, one process per GPU: cuBLAS GEMMs + NCCL all_gather_into_tensor / all_reduce."""

    def __init__(self, cfg: TPConfig, rank: int, world: int, device, scatter: bool = False):
        self.cfg, self.rank, self.world = cfg, rank, world
        self.scatter = bool(scatter) and world > 1   # reduce_scatter_tensor instead of all_reduce
        if not cfg.plain:
            raise ValueError("the baseline has no positions, head norms, windows or grouped heads")
        T, H, I = cfg.tokens, cfg.hidden, cfg.intermediate
        self.heads_local = cfg.n_heads // world
        self.ts = T // world
        self.w = []
        for layer in range(cfg.n_layers):
            full = layer_weights(cfg, layer, device)
            self.w.append(shard_weights(full, cfg, rank, world))
            del full
        bf = dict(dtype=torch.bfloat16, device=device)
        self.xn = torch.empty((self.ts, H), **bf)
        self.full = torch.empty((T, H), **bf)
        self.qkv = torch.empty((T, 3 * H // world), **bf)
        self.attn = torch.empty((T, H // world), **bf)
        self.part = torch.empty((T, H), **bf)
        self.kept = torch.empty((self.ts, H), **bf)
        self.gu = torch.empty((T, 2 * I // world), **bf)
        self.h = torch.empty((T, I // world), **bf)

    def forward(self, x_shard: torch.Tensor, timers=None) -> torch.Tensor:
        import torch.distributed as dist
        cfg = self.cfg
        tick = timers if timers is not None else (lambda name: None)
        rows = slice(self.rank * self.ts, (self.rank + 1) * self.ts)

        def gather(t):
            if self.world > 1:
                dist.all_gather_into_tensor(self.full, t)
            else:
                self.full.copy_(t)

        def reduce(t):
            """Sum over ranks; returns this rank's token rows of the sum."""
            if self.scatter:
                dist.reduce_scatter_tensor(self.kept, t)
                return self.kept
            if self.world > 1:
                dist.all_reduce(t)
            return t[rows]
        for w in self.w:
            tick("norm")
            E.rmsnorm(x_shard, w["norm1"], self.xn, cfg.eps)
            tick("qkv_ag_gemm")
            gather(self.xn)
            torch.matmul(self.full, w["wqkv"].t(), out=self.qkv)
            tick("attention")
            attention(self.qkv, cfg, self.heads_local, self.attn)
            tick("o_gemm_ar")
            torch.matmul(self.attn, w["wo"].t(), out=self.part)
            kept = reduce(self.part)
            tick("norm")
            E.residual_add(x_shard, kept)
            E.rmsnorm(x_shard, w["norm2"], self.xn, cfg.eps)
            tick("gu_ag_gemm")
            gather(self.xn)
            torch.matmul(self.full, w["wgu"].t(), out=self.gu)
            tick("swiglu")
            E.swiglu(self.gu, self.h)
            tick("down_gemm_ar")
            torch.matmul(self.h, w["wd"].t(), out=self.part)
            kept = reduce(self.part)
            tick("norm")
            E.residual_add(x_shard, kept)
        tick("end")
        return x_shard


def reference_forward(x: torch.Tensor, cfg: TPConfig) -> torch.Tensor:
    """Unsharded fp32 oracle: x [T, H] (any float dtype) -> [T, H] fp32, with the same bf16 weights."""
    dev = x.device
    x = x.float().clone()
    B, S, nh, kv, d = cfg.batch, cfg.seq, cfg.n_heads, cfg.kv_heads, cfg.head_dim
    at = torch.arange(S, device=dev)
    seen = (at <= at[:, None]) & ((at > at[:, None] - cfg.window) | (at < cfg.sinks)) if cfg.window else None

    def norm(t, w):
        return t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + cfg.eps) * w.float()

    def rotate(t):
        rot = cfg.rotary_dim or d
        angle = at.double()[:, None] * cfg.rope_theta ** (-torch.arange(0, rot, 2, device=dev).double() / rot)
        c, s = angle.cos().float(), angle.sin().float()
        i = torch.arange(0, rot, 2, device=dev) if cfg.interleaved else torch.arange(rot // 2, device=dev)
        j = i + 1 if cfg.interleaved else i + rot // 2
        y = t.clone()
        y[..., i], y[..., j] = t[..., i] * c - t[..., j] * s, t[..., j] * c + t[..., i] * s
        return y
    for layer in range(cfg.n_layers):
        w = layer_weights(cfg, layer, dev)
        xn = norm(x, w["norm1"])
        q = (xn @ w["wq"].float().t()).view(B, S, nh, d).transpose(1, 2)
        k = (xn @ w["wk"].float().t()).view(B, S, kv, d).transpose(1, 2)
        v = (xn @ w["wv"].float().t()).view(B, S, kv, d).transpose(1, 2)
        if cfg.qk_norm:
            q, k = norm(q, w["q_norm"]), norm(k, w["k_norm"])
        if cfg.rope_theta:
            q, k = rotate(q), rotate(k)
        k, v = (t.repeat_interleave(nh // kv, 1) for t in (k, v))
        a = F.scaled_dot_product_attention(q, k, v, attn_mask=seen, is_causal=seen is None).transpose(1, 2).reshape(B * S, nh * d)
        x = x + a @ w["wo"].float().t()
        xn = norm(x, w["norm2"])
        hidden = F.silu(xn @ w["wg"].float().t()) * (xn @ w["wu"].float().t())
        x = x + hidden @ w["wd"].float().t()
    return x
