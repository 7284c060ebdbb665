"""Grouped-query attention over the paged cache.

One product gives q, k and v of a token (the reference keeps Wq, Wk, Wv in one
buffer for the same reason, src/model/attn.cuh:113-118, 235-243); queries and keys
are rotated and keys and values stored into the cache in one kernel; attention
runs over the cache, which then already holds this step's tokens; the output
projection follows (src/model/attn.cuh:185-229).  With ``sparse`` given, queries that
see more than ``dense_len`` keys attend only to selected key blocks (InfLLM-v2,
src/model/minicpm4/minicpm4_attn.cuh:95-202); that rule is per query, so it does not
depend on how tokens are cut into steps.
"""
from __future__ import annotations

import math
from typing import Any, Dict, Mapping, Optional

import torch

from .base import KV4_HEAD_DIMS, MIXERS, POSITIONS, CacheNeeds, Mixer, PartSpec, WeightSpec, build_part


@MIXERS.register("gqa_attention")
class GroupedQueryAttention(Mixer):
    @property
    def recordable_prompt(self) -> bool:
        return bool(self.position.recordable_prompt)

    def __init__(self, ops, hidden_size: int, n_heads: int, n_kv_heads: int, head_dim: int,
                 position: PartSpec, window: Optional[int] = None, sparse: Optional[Mapping[str, int]] = None,
                 softmax_scale: Optional[float] = None, position_name: str = "", cache_bits: int = 16):
        """``cache_bits`` 4: keys and values are held in 4 bits (``Ops.rope_store_kv4``).  ``position_name``: infix of the position part's own tensors below this part's prefix (an encoding with
        learned tables declares them in its ``weight_specs``; the rotary encodings have none)."""
        super().__init__(ops)
        if window and sparse:
            # a windowed lane gives pages back that the block selection (leading blocks, chosen far blocks, the
            # scores over all pooled keys) would still follow
            raise ValueError("gqa_attention takes a window or a sparse configuration, not both")
        if n_heads % n_kv_heads:
            raise ValueError(f"{n_heads} heads cannot be grouped over {n_kv_heads} key-value heads")
        if head_dim % 16 or head_dim > 256:
            raise ValueError(f"head_dim {head_dim}: the attention kernels take multiples of 16 up to 256")
        if cache_bits not in (4, 16):
            raise ValueError(f"cache_bits is 4 or 16, got {cache_bits}")
        if cache_bits == 4 and (sparse or head_dim not in KV4_HEAD_DIMS):
            raise ValueError(f"a cache in 4 bits takes dense attention with head sizes {KV4_HEAD_DIMS}"
                             + (", not a sparse configuration" if sparse else f", not {head_dim}"))
        self.four_bits = cache_bits == 4
        self.hidden_size, self.n_heads, self.n_kv, self.d = int(hidden_size), int(n_heads), int(n_kv_heads), int(head_dim)
        self.window = int(window) if window else 0
        self.sparse = dict(sparse) if sparse else None
        self.scale = float(softmax_scale) if softmax_scale is not None else 1.0 / math.sqrt(self.d)
        self.position = build_part(POSITIONS, position, ops)
        self.position_name = str(position_name)
        self.w_qkv: Optional[torch.Tensor] = None
        self.w_o: Optional[torch.Tensor] = None

    # ---- weights ----
    def weight_specs(self) -> Dict[str, WeightSpec]:
        h, d = self.hidden_size, self.d
        specs = {
            "q_proj.weight": WeightSpec((self.n_heads * d, h)),
            "k_proj.weight": WeightSpec((self.n_kv * d, h)),
            "v_proj.weight": WeightSpec((self.n_kv * d, h)),
            "o_proj.weight": WeightSpec((h, self.n_heads * d)),
        }
        for name, spec in self.position.weight_specs().items():
            specs[self.position_name + name] = spec
        return specs

    def load_weights(self, tensors: Dict[str, torch.Tensor]) -> None:
        own = self.position.weight_specs()
        if own:
            self.position.load_weights({n: tensors[self.position_name + n] for n in own})
        self.w_qkv = self.ops.keep(torch.cat([tensors["q_proj.weight"], tensors["k_proj.weight"], tensors["v_proj.weight"]],
                                             dim=0).contiguous())
        self.w_o = self.ops.keep(tensors["o_proj.weight"].contiguous())

    def weight_bytes(self) -> int:
        return (self.w_qkv.numel() + self.w_o.numel()) * self.w_qkv.element_size()

    # ---- cache ----
    def cache_needs(self) -> CacheNeeds:
        stride = self.sparse["kernel_stride"] if self.sparse else 0
        kernel = self.sparse["kernel_size"] if self.sparse else 0
        return CacheNeeds(kv_heads=self.n_kv, head_dim=self.d, window=self.window or None,
                          pooled_stride=stride, pooled_kernel=kernel, bits=4 if self.four_bits else 0)

    def cache_bytes_read(self, kv_len: int) -> int:
        keys = min(kv_len, self.window) if self.window else kv_len
        pooled = 0
        if self.sparse is not None and kv_len > self.sparse.get("dense_len", 0):
            # the leading and chosen blocks (topk of them) and the local window, and every visible pooled key (fp32)
            sp = self.sparse
            blocks = sp["topk"] + sp["window_size"] // sp["block_size"]
            keys = min(kv_len, blocks * sp["block_size"])
            pooled = max(0, (kv_len - sp["kernel_size"]) // sp["kernel_stride"] + 1) * self.n_kv * self.d * 4
        if self.four_bits:
            return keys * self.n_kv * (self.d + 16)
        return 2 * keys * self.n_kv * self.d * self.ops.element_size + pooled

    # ---- forward ----
    def forward(self, ctx, y: torch.Tensor, lane, writes_cache: bool) -> torch.Tensor:
        ops = self.ops
        if lane.n_pages:
            ops.set_page_limit(lane.n_pages)             # the checked build's kernels compare page numbers with it
        qkv = ops.linear(y, self.w_qkv)
        inv_freq, magnitude, rot_dim = self.position.rotary() or (None, 1.0, -1)
        k_cache, v_cache = lane.k, lane.v
        if rot_dim < 0:
            # an encoding that is not a rotation of pairs transforms q and k itself
            row = qkv.view(ctx.n_tokens, self.n_heads + 2 * self.n_kv, self.d)
            self.position.apply(ctx, row[:, :self.n_heads], row[:, self.n_heads:self.n_heads + self.n_kv])
            inv_freq, magnitude, rot_dim = None, 1.0, 0
        if self.four_bits:
            q = ops.rope_store_kv4(qkv, self.n_heads, self.n_kv, self.d, ctx.positions, ctx.token_seq, ctx.slot_dev, lane.page_table,
                                   lane.records if writes_cache else None, inv_freq, magnitude, rot_dim)
            prompt = {} if ctx.is_decode else dict(cu_q=ctx.cu_q, tiles=ctx.q_tiles, longest=ctx.max_kv_len)
            out = ops.kv4_attention(q, lane.records, ctx.kv_len_dev, ctx.slot_dev, lane.page_table, self.n_kv, self.scale, self.window, **prompt)
            return ops.linear(out, self.w_o)
        if rot_dim >= 0 and ops.fused_decode_ok(ctx, self.d, rot_dim, self.window, self.sparse):
            # one token per sequence: the attention kernel rotates, stores the new key and value, and attends
            out = ops.decode_attention_rope(qkv, lane, ctx.kv_len_dev, ctx.slot_dev, self.n_heads, self.n_kv, self.d,
                                            self.scale, inv_freq if rot_dim else None, magnitude, writes_cache)
            return ops.linear(out, self.w_o)
        q = ops.rope_store(qkv, self.n_heads, self.n_kv, self.d, ctx.positions, ctx.token_seq, ctx.slot_dev,
                           lane.page_table, k_cache if writes_cache else None, v_cache if writes_cache else None,
                           inv_freq, magnitude, rot_dim)
        block_list, block_size = None, 0
        if self.sparse is not None:
            if writes_cache:
                ops.pool_keys(ctx, lane, self.n_kv, self.d, self.sparse["kernel_size"], self.sparse["kernel_stride"])
            if ctx.max_kv_len > self.sparse.get("dense_len", 0):      # in a recorded step an upper bound: still the right test
                block_list, block_size = ops.select_blocks(ctx, q, lane, self.n_kv, self.scale, self.sparse)
                taps = ctx.extras.get("taps")
                if taps is not None and not ctx.captured:
                    # a caller that wants to see the choice (tests do): lane, the step's slots, and per token its
                    # sequence, position and block lists
                    taps.setdefault("block_lists", []).append(
                        (lane.index, list(ctx.slots), ctx.token_seq.clone(), ctx.positions.clone(), block_list.clone()))
        out = ops.attention(ctx, q, lane, self.n_kv, self.scale, self.window, block_list, block_size)
        return ops.linear(out, self.w_o)


@MIXERS.register("sink_window_attention")
class SinkWindowAttention(Mixer):
    """Grouped-query softmax attention over the paged cache with biased projections, unit-rms queries and keys, capped
    scores, a sliding window and a sink:

        q = Wq h + bq,  k = Wk h + bk,  v = Wv h + bv           (q, k heads of ``head_dim`` channels, v of ``value_dim``)
        q <- q / sqrt(mean(q^2) + eps) * g_q,  k likewise with g_k                     (``row_norm``: over a token's whole q row and
                                                 whole k row, all heads at once, tensors ``names["q_norm"]``, ``names["k_norm"]``)
        q, k <- position(q, k);   q, k <- x / sqrt(mean(x^2) + eps) per head          (``unit_rms``; no weight)
        s(i, j) = q_i . k_j * softmax_scale;   s <- softcap * tanh(s / softcap)        (``softcap`` > 0)
        j is seen by i when 0 <= i - j < window                                        (``window``; None: all j <= i)
            or j < keep_first and j <= i                                               (``keep_first``: tokens a window keeps)
        p_j = exp(s_j) / (exp(b_h) + sum_j' exp(s_j'))      (``sink``: a further key without a value, of score b_h = 0, or with
                                                             "learned" a number per head, tensor ``names["sink"]``; else plain)
        o_h = sum_j p_j v_kv(h)(j);   o_h <- o_h * sigmoid(Wg h)_h                     (``gate``: ``names["gate"]`` [heads, hidden])
        out = Wo [o_0 | o_1 | ...]

    With ``own_kv`` False the layer has no key and value projections: it reads the lane another layer of equal head
    counts and rotation wrote (keys as cached, after rotation and norm), with its own queries, window, cap and scale.
    ``biases``: which of "q", "k", "v" have one (tensor name + ``names["bias"]``).  Biases, norms, rotation, the unit rms,
    scores and weights are 32-bit; keys and values live in the cache in the compute dtype.
    """

    DEFAULT_NAMES = {"q": "q", "k": "k", "v": "v", "o": "o", "bias": ".b", "sink": "sink", "gate": "g",
                     "q_norm": "q.norm", "k_norm": "k.norm"}

    @property
    def recordable_prompt(self) -> bool:
        return bool(self.position.recordable_prompt)

    def __init__(self, ops, hidden_size: int, n_heads: int, n_kv_heads: int, head_dim: int, value_dim: int,
                 softmax_scale: float, position: PartSpec, eps: float, window: Optional[int] = None, softcap: float = 0.0,
                 sink=True, unit_rms: bool = True, biases=("q", "k", "v"), own_kv: bool = True, names=None,
                 keep_first: int = 0, gate: bool = False, row_norm: bool = False):
        super().__init__(ops)
        if n_heads % n_kv_heads:
            raise ValueError(f"{n_heads} heads cannot be grouped over {n_kv_heads} key-value heads")
        if head_dim > 256 or value_dim > 256:
            raise ValueError("sink_window_attention: the kernels take heads of up to 256 channels")
        self.hidden_size, self.n_heads, self.n_kv = int(hidden_size), int(n_heads), int(n_kv_heads)
        self.d, self.dv, self.scale, self.eps = int(head_dim), int(value_dim), float(softmax_scale), float(eps)
        self.window = int(window) if window else 0
        self.softcap, self.sink, self.unit_rms, self.own_kv = float(softcap or 0.0), bool(sink), bool(unit_rms), bool(own_kv)
        self.learned_sink = sink == "learned"
        self.keep_first = int(keep_first or 0) if self.window else 0
        self.gate = bool(gate)
        self.row_norm = bool(row_norm)
        if self.row_norm and self.unit_rms:
            raise ValueError("sink_window_attention: a norm over the whole rows and a unit rms per head exclude each other")
        self.norms = None
        self.sinks: Optional[torch.Tensor] = None
        self.biases = tuple(b for b in ("q", "k", "v") if b in tuple(biases) and (b == "q" or self.own_kv))
        self.position = build_part(POSITIONS, position, ops)
        self.names = dict(self.DEFAULT_NAMES, **(dict(names) if names else {}))
        self.bias = {"q": None, "k": None, "v": None}

    def _projections(self):
        G, d, dv = self.n_kv, self.d, self.dv
        return [("q", self.n_heads * d)] + ([("k", G * d), ("v", G * dv)] if self.own_kv else [])

    def weight_specs(self) -> Dict[str, WeightSpec]:
        n, W = self.names, self.hidden_size
        specs = {n["o"]: WeightSpec((W, self.n_heads * self.dv))}
        if self.learned_sink:
            specs[n["sink"]] = WeightSpec((self.n_heads,), "vector")
        if self.gate:
            specs[n["gate"]] = WeightSpec((self.n_heads, W))
        if self.row_norm:
            specs[n["q_norm"]] = WeightSpec((self.n_heads * self.d,), "vector")
            if self.own_kv:
                specs[n["k_norm"]] = WeightSpec((self.n_kv * self.d,), "vector")
        for which, rows in self._projections():
            specs[n[which]] = WeightSpec((rows, W))
            if which in self.biases:
                specs[n[which] + n["bias"]] = WeightSpec((rows,), "vector")
        return specs

    def load_weights(self, tensors: Dict[str, torch.Tensor]) -> None:
        n = self.names
        rows = [tensors[n[which]] for which, _ in self._projections()] + ([tensors[n["gate"]]] if self.gate else [])
        self.w_in = self.ops.keep(torch.cat(rows, dim=0).contiguous())       # one product: q (k, v) and the gates' logits
        self.w_o = self.ops.keep(tensors[n["o"]].contiguous())
        if self.learned_sink:
            self.sinks = self.ops.keep(tensors[n["sink"]].float().contiguous())
        if self.row_norm:
            self.norms = (self.ops.keep(tensors[n["q_norm"]].float().contiguous()),
                          self.ops.keep(tensors[n["k_norm"]].float().contiguous()) if self.own_kv else None)
        for which in self.biases:
            self.bias[which] = self.ops.keep(tensors[n[which] + n["bias"]].float().contiguous())

    def weight_bytes(self) -> int:
        return (self.w_in.numel() + self.w_o.numel()) * self.w_in.element_size() + \
            4 * sum(b.numel() for b in (*self.bias.values(), *(self.norms or ())) if b is not None)

    def cache_needs(self) -> CacheNeeds:
        return CacheNeeds(kv_heads=self.n_kv, head_dim=self.d, window=self.window or None,
                          value_dim=self.dv if self.dv != self.d else 0, keep_first=self.keep_first)

    def cache_bytes_read(self, kv_len: int) -> int:
        keys = min(kv_len, self.window + self.keep_first) if self.window else kv_len
        return keys * self.n_kv * (self.d + self.dv) * self.ops.element_size

    def forward(self, ctx, y: torch.Tensor, lane, writes_cache: bool) -> torch.Tensor:
        ops = self.ops
        if writes_cache != self.own_kv:
            raise ValueError("sink_window_attention: a layer with projections of its own writes its lane, one without reads "
                             "another's (the schedule and the layer disagree)")
        if lane.k is not None:
            ops.set_page_limit(lane.k.shape[0])
        rot = self.position.rotary()
        if rot is None or rot[1] != 1.0:
            raise ValueError("sink_window_attention takes a rotation of pairs without a magnitude factor, or no position encoding")
        inv_freq, _, rot_dim = rot
        proj = ops.linear(y, self.w_in, out_f32=True)
        H = self.n_heads
        q = ops.qk_prepare_store(ctx, proj, lane, H, self.n_kv, self.d, self.dv,
                                 (self.bias["q"], self.bias["k"], self.bias["v"]), inv_freq if rot_dim else None, rot_dim,
                                 self.unit_rms, self.eps, has_kv=self.own_kv, adjacent=bool(getattr(self.position, "adjacent", False)),
                                 extra_cols=H if self.gate else 0, norms=self.norms)
        gate = proj[:, proj.shape[1] - H:] if self.gate else None
        out = ops.sink_attention(ctx, q, lane, self.n_kv, self.dv, self.scale, self.window, self.softcap, self.sink,
                                 keep_first=self.keep_first, sinks=self.sinks, gate=gate)
        return ops.linear(out, self.w_o)
