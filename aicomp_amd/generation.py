"""Generation driver over the paged path: the caller of the attention operator.

Mirrors ``ScheduleGeneration`` of the reference
(opt_prime/opt_prime/schedule_infer.py:341-449): ``prefill`` runs the prompt and
returns the logits of the last position, ``decode_step`` runs one token per
sequence, ``clear_cache`` resets.  Differences, all on purpose:

* every sequence has its own length and position (the reference shares one scalar
  position, ``schedule_infer.py:425-430``), so prompts of different lengths and
  continuous batching work;
* the next-step input may be ``[B]`` or ``[B, 1]``: it is flattened to one token per
  sequence.  The reference's loop builds it with ``next_token.unsqueeze(0)``
  (opt_prime/opt_prime/inference.py:1041-1043), i.e. ``[1, B]``, which only has the
  right shape for batch 1;
* the model is called token-major: ``model(input_ids [T], positions [T]) ->
  logits [T, V]``, its attention layers calling ``PagedAttentionBackend.attend``.

``PagedAttentionBackend`` owns one K and one V pool per layer and runs, per layer and
step, the rotary embedding fused with the append followed by the chunked-prefill
kernel on the prompt-chunk rows and the decode kernel on the one-token rows; a small
step of one-token rows alone is one launch (``ops.rope_paged_decode_attn``).  A layer may norm its query and key
heads (``set_head_norm``) and score by a rule (``set_score_rule``: a cap, a bias by distance, a window); its steps
then run ``ops.qk_norm_rope_kv_append`` and the ``ops.paged_score_*`` calls.
"""
from __future__ import annotations

import math
from typing import Callable, Dict, List, Optional, Sequence

import numpy as np
import torch

from . import ops
from .block_manager import StepPlan, StepPlanner


class PagedAttentionBackend:
    """Per-layer paged K/V pools plus the per-step attention call of a decoder layer.

    ``inv_freq`` (the rotary module's buffer, compiler_fx/modeling_llama.py:130-132) switches
    the rotary embedding on: ``attend`` then takes Q/K as projected and rotates them itself.
    Without it Q/K must arrive rotated.  With fewer than ``head_dim / 2`` frequencies the rest of each head is not rotated;
    ``interleaved`` rotates neighbours instead of halves (both are computed in float32 and rounded once, where the
    rotation of whole heads by halves repeats the roundings of the reference's eager evaluation).
    """

    def __init__(self, num_layers: int, num_blocks: int, num_kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.bfloat16, device="cuda", kv_dtype: Optional[torch.dtype] = None,
                 inv_freq: Optional[torch.Tensor] = None, max_positions: int = 8192,
                 attention_scaling: float = 1.0, scale: Optional[float] = None, block_size: int = 16,
                 interleaved: bool = False) -> None:
        self.device = torch.device(device)
        self.dtype = dtype
        kv_dtype = kv_dtype or dtype
        shape = (num_blocks, num_kv_heads, block_size, head_dim)
        self.k_pools = [torch.zeros(shape, dtype=kv_dtype, device=self.device) for _ in range(num_layers)]
        self.v_pools = [torch.zeros(shape, dtype=kv_dtype, device=self.device) for _ in range(num_layers)]
        self.k_scales: List[Optional[torch.Tensor]] = [None] * num_layers
        self.v_scales: List[Optional[torch.Tensor]] = [None] * num_layers
        self.scale = 1.0 / math.sqrt(head_dim) if scale is None else scale
        self.cos = self.sin = None
        self.interleaved = bool(interleaved)
        # float32 tables of a layer that norms its heads, or of every layer where the rotation is not that of whole heads by halves
        self._pair_tables = None
        self._pairs_from = None if inv_freq is None else (inv_freq, max_positions, attention_scaling)
        self._pairs_only = inv_freq is not None and (self.interleaved or 2 * inv_freq.numel() != head_dim)
        if inv_freq is not None and not self._pairs_only:
            self.cos, self.sin = ops.rotary_tables(inv_freq, max_positions, dtype, attention_scaling, self.device)
        if self._pairs_only:
            self._pairs()
        self._norms: Dict[int, tuple] = {}
        self._rules: Dict[int, dict] = {}
        self.plan: Optional[StepPlan] = None
        self.first_keys: Optional[torch.Tensor] = None
        self.prefix_lens: Optional[torch.Tensor] = None

    def _pairs(self):
        if self._pair_tables is None and self._pairs_from is not None:
            inv_freq, positions, scaling = self._pairs_from
            self._pair_tables = ops.rotary_pair_tables(inv_freq, positions, scaling, self.device)
        return self._pair_tables or (None, None)

    @property
    def num_positions(self) -> Optional[int]:
        """Rows of the rotary tables, ``None`` without them."""
        return None if self._pairs_from is None else int(self._pairs_from[1])

    def set_head_norm(self, layer_idx: int, q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor],
                      eps: float = 1e-6) -> None:
        """RMS norm of every query and key head of a layer before the rotation, weights ``[D]`` (``None``: not that one)."""
        f32 = lambda w: None if w is None else w.to(self.device, torch.float32).contiguous()
        self._norms[layer_idx] = (f32(q_weight), f32(k_weight), float(eps))
        self._pairs()                                  # (built here, not in the first step)

    def set_score_rule(self, layer_idx: int, softcap: float = 0.0, slopes: Optional[torch.Tensor] = None, window: int = 0) -> None:
        """Scores of a layer: capped by a tanh, less ``slopes[h]`` times the distance, over the last ``window`` keys."""
        if softcap < 0 or window < 0:
            raise ValueError(f"softcap and window must not be negative, got {softcap}, {window}")
        self._rules[layer_idx] = dict(softcap=float(softcap), window=int(window),
                                      slopes=None if slopes is None else slopes.to(self.device, torch.float32).contiguous())

    def copy_blocks(self, pairs) -> None:
        """Blocks copied in every layer's pools: what ``StepPlanner.fork`` and ``compact`` return."""
        pairs = torch.from_numpy(np.ascontiguousarray(pairs, dtype=np.int64))
        if pairs.shape[0]:
            ops.copy_blocks(self.k_pools + self.v_pools, pairs)

    def set_scales(self, layer_idx: int, k_scale: torch.Tensor, v_scale: torch.Tensor) -> None:
        """Per-KV-head dequantisation scales of an fp8 pool."""
        self.k_scales[layer_idx] = k_scale.to(self.device, torch.float32).contiguous()
        self.v_scales[layer_idx] = v_scale.to(self.device, torch.float32).contiguous()

    def begin_step(self, plan: StepPlan, first_keys: Optional[torch.Tensor] = None, prefix_lens=None) -> None:
        """``first_keys [T]`` int32: the first key that each row of the step sees (packed documents); ``prefix_lens [S]`` int32: the
        part at the start of each sequence that all its rows see, on the host (a sequence, an array, a CPU tensor; a tensor on the
        device is read back, which waits for it).  Both hold for every layer of the step.

        All rows of a prefix see each other, so it has to be ingested by one step: one that reaches beyond its sequence's
        context in this step is refused (``StepPlanner.add_request(..., prefix_len=...)`` keeps it in one chunk)."""
        if prefix_lens is not None:
            if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("begin_step with prefix_lens goes before the recording of a step: their values are looked at")
            lens = torch.as_tensor(prefix_lens)
            host = lens.cpu().numpy()
            if lens.shape != (plan.num_seqs,) or host.dtype.kind not in "iu":
                raise ValueError(f"prefix_lens must be {plan.num_seqs} whole numbers, one per sequence of the step; got "
                                 f"{host.dtype} {tuple(lens.shape)}")
            beyond = np.flatnonzero(host > plan.host_context_lens)
            if beyond.size:
                r = int(beyond[0])
                raise ValueError(f"sequence {plan.seq_ids[r]!r}: its prefix of {int(host[r])} tokens is not in this step, which ends at "
                                 f"{int(plan.host_context_lens[r])}; a prefix is ingested in one chunk "
                                 f"(StepPlanner.add_request(..., prefix_len={int(host[r])}))")
            prefix_lens = lens.to(self.device, torch.int32).contiguous()
        self.plan, self.first_keys, self.prefix_lens = plan, first_keys, prefix_lens

    def _score_attend(self, layer_idx: int, out: torch.Tensor, q: torch.Tensor) -> torch.Tensor:
        """Attention of a step by the layer's rule: its rows are in the pools, ``q`` is rotated."""
        plan, kp, vp = self.plan, self.k_pools[layer_idx], self.v_pools[layer_idx]
        ks, vs = self.k_scales[layer_idx], self.v_scales[layer_idx]
        rule = self._rules.get(layer_idx, {})
        npre, S, t = plan.num_prefill_seqs, plan.num_seqs, plan.num_prefill_tokens
        first, prefix = self.first_keys, self.prefix_lens
        # (a recorded launch is sized for the whole table: the lengths of its replays may grow)
        sized = not (q.is_cuda and torch.cuda.is_current_stream_capturing())
        if npre:
            ops.paged_score_prefill_attn(out[:t], q[:t], kp, vp, plan.block_table[:npre], plan.context_lens[:npre],
                                         plan.cu_q_lens[:npre + 1], self.scale, max_q_len=plan.max_q_len,
                                         first_keys=None if first is None else first[:t],
                                         prefix_lens=None if prefix is None else prefix[:npre], k_scale=ks, v_scale=vs,
                                         longest_context=int(plan.host_context_lens[:npre].max()) if sized else 0, **rule)
        if S > npre:
            ops.paged_score_decode_attn(out[t:], q[t:], kp, vp, plan.block_table[npre:], plan.context_lens[npre:], self.scale,
                                        first_keys=None if first is None else first[t:], k_scale=ks, v_scale=vs,
                                        longest_context=int(plan.host_context_lens[npre:].max()) if sized else 0, **rule)
        return out

    def attend(self, layer_idx: int, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor) -> torch.Tensor:
        """``query [T, Hq, D]``, ``key`` / ``value [T, Hkv, D]`` in the plan's row order -> ``[T, Hq, D]``."""
        plan = self.plan
        if plan is None:
            raise RuntimeError("PagedAttentionBackend.attend called outside a step (begin_step first)")
        kp, vp = self.k_pools[layer_idx], self.v_pools[layer_idx]
        ks, vs = self.k_scales[layer_idx], self.v_scales[layer_idx]
        norm = self._norms.get(layer_idx)
        ruled = layer_idx in self._rules or self.first_keys is not None or self.prefix_lens is not None
        if ruled or norm is not None or self._pairs_only:
            q = torch.empty(query.shape, dtype=query.dtype, device=query.device)
            if norm is not None or self._pairs_only:
                q_weight, k_weight, eps = norm or (None, None, 0.0)
                cos, sin = self._pairs()
                ops.qk_norm_rope_kv_append(query, key, value, q_weight, k_weight, cos, sin, plan.positions, kp, vp,
                                           plan.slot_mapping, eps, self.interleaved, ks, vs, query_out=q)
            elif self.cos is not None:
                ops.rope_kv_append(query, key, value, self.cos, self.sin, plan.positions, kp, vp, plan.slot_mapping, ks, vs,
                                   query_out=q)
            else:
                ops.kv_append(key, value, kp, vp, plan.slot_mapping, ks, vs)
                q = query.contiguous()
            out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
            return self._score_attend(layer_idx, out, q) if ruled else self._attend(layer_idx, out, q)
        if self.cos is not None and plan.num_prefill_seqs == 0:          # one token per sequence: one launch, if it can be
            out = ops.rope_paged_decode_attn(query, key, value, self.cos, self.sin, plan.positions, kp, vp,
                                             plan.slot_mapping, plan.block_table, plan.context_lens,
                                             plan.host_context_lens, self.scale, ks, vs, plan.host_slot_mapping,
                                             plan.host_block_table)
            if out is not None:
                return out
        out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
        if self.cos is None:
            from .block_manager import paged_attention_step
            return paged_attention_step(plan, out, query.contiguous(), key, value, kp, vp, self.scale, ks, vs)
        q = torch.empty(query.shape, dtype=query.dtype, device=query.device)
        ops.rope_kv_append(query, key, value, self.cos, self.sin, plan.positions, kp, vp, plan.slot_mapping,
                           ks, vs, query_out=q)
        return self._attend(layer_idx, out, q)

    def _attend(self, layer_idx: int, out: torch.Tensor, q: torch.Tensor) -> torch.Tensor:
        """Causal attention of a step whose rows are in the pools."""
        plan, kp, vp = self.plan, self.k_pools[layer_idx], self.v_pools[layer_idx]
        ks, vs = self.k_scales[layer_idx], self.v_scales[layer_idx]
        npre, S, t_pre = plan.num_prefill_seqs, plan.num_seqs, plan.num_prefill_tokens
        items = plan.launch_items(q, kp)
        if items is not None:                      # mixed step: chunks and decode rows in one launch
            return ops.paged_prefill_attn(out, q, kp, vp, plan.block_table, plan.context_lens, plan.cu_q_lens,
                                          self.scale, max_q_len=plan.launch_q_len(q.shape[1], kp.shape[1]), k_scale=ks,
                                          v_scale=vs, items=items)
        if plan.only_chunks and t_pre == q.shape[0]:         # chunks alone, rows alone: the plan's tensors as they are
            return ops.append_prefill_attn(out, q, None, None, kp, vp, None, plan.block_table, plan.context_lens,
                                           plan.cu_q_lens, self.scale, plan.max_q_len, ks, vs, plan.prefill_items(q, kp),
                                           plan.host_context_lens)
        if S and npre == 0:
            return ops.paged_decode_attn(out, q, kp, vp, plan.block_table, plan.context_lens, self.scale, ks, vs)
        if npre and S > npre:
            return ops.chunks_and_rows_attn(out, q, None, None, kp, vp, None, plan.block_table, plan.context_lens,
                                            plan.cu_q_lens, self.scale, plan.max_q_len, npre, t_pre, ks, vs,
                                            plan.prefill_items(q, kp), plan.few_chunk_lens(q.shape[1], kp.shape[1]))
        if npre:
            ops.paged_prefill_attn(out[:t_pre], q[:t_pre], kp, vp, plan.block_table[:npre], plan.context_lens[:npre],
                                   plan.cu_q_lens[:npre + 1], self.scale, max_q_len=plan.max_q_len,
                                   k_scale=ks, v_scale=vs, items=plan.prefill_items(q, kp))
        return out


class ScheduleGeneration:
    """``prefill`` / ``decode_step`` / ``clear_cache`` over a token-major model and a planner."""

    def __init__(self, model: Callable[[torch.Tensor, torch.Tensor], torch.Tensor],
                 backend: PagedAttentionBackend, planner: StepPlanner) -> None:
        # a token whose position has no row in the rotary tables would be left unrotated and
        # unstored by the fused rotary + append launch: refuse the combination up front
        cos, positions = getattr(backend, "cos", None), getattr(backend, "num_positions", None)
        if positions is None and cos is not None:
            positions = cos.shape[0]
        if positions is not None and planner.max_seq_len > positions:
            raise ValueError(f"the planner admits sequences of {planner.max_seq_len} tokens but the backend's "
                             f"rotary tables hold {positions} positions (max_positions)")
        self.model = model
        self.backend = backend
        self.planner = planner
        self._batch: List[object] = []
        self._offset: Dict[object, int] = {}

    # one planner step: returns {seq_id: logits row of its last new token}
    @torch.no_grad()
    def _step(self, tokens_of: Dict[object, torch.Tensor], decode=None) -> Dict[object, torch.Tensor]:
        plan = self.planner.schedule(decode)
        if plan is None:
            return {}
        if plan.preempted:
            raise RuntimeError(f"pool too small for this batch: sequences {plan.preempted} were preempted")
        cu = plan.host_cu_q_lens
        pieces = []
        for r, sid in enumerate(plan.seq_ids):
            n = int(plan.new_lens[r])
            start = int(plan.host_positions[cu[r]]) - self._offset.get(sid, 0)
            pieces.append(tokens_of[sid][start:start + n])
        ids = torch.cat(pieces).to(self.backend.device)
        self.backend.begin_step(plan)
        logits = self.model(ids, plan.positions)
        last = torch.as_tensor(cu[1:] - 1, dtype=torch.int64, device=logits.device)
        rows = logits.index_select(0, last)
        return {sid: rows[r] for r, sid in enumerate(plan.seq_ids)}

    @torch.no_grad()
    def prefill(self, input_ids: torch.Tensor, position_ids: Optional[torch.Tensor] = None,
                prompt_lens: Optional[Sequence[int]] = None) -> torch.Tensor:
        """Ingest the prompts ``input_ids [B, S]`` (right-padded when ``prompt_lens`` gives shorter
        lengths) and return the logits after each prompt's last token, ``[B, V]``
        (schedule_infer.py:363-407).  ``position_ids`` is accepted for signature compatibility;
        positions always run from 0 per sequence."""
        if input_ids.dim() == 1:
            input_ids = input_ids[None, :]
        B, S = input_ids.shape
        lens = [S] * B if prompt_lens is None else [int(n) for n in prompt_lens]
        self.clear_cache()
        self._offset = {}
        toks = {}
        for b in range(B):
            self.planner.add_request(b, lens[b])
            toks[b] = input_ids[b, :lens[b]]
        self._batch = list(range(B))
        final: Dict[object, torch.Tensor] = {}
        while len(final) < B:
            got = self._step(toks, decode=())      # nobody decodes until every prompt is in
            if not got:
                raise RuntimeError("planner made no progress during prefill")
            for sid, row in got.items():
                if self.planner.context_len(sid) == lens[sid]:
                    final[sid] = row
        return torch.stack([final[b] for b in range(B)])

    @torch.no_grad()
    def decode_step(self, input_token: torch.Tensor, position=None) -> torch.Tensor:
        """One token per sequence: ``input_token`` ``[B]``, ``[B, 1]`` (or the reference's ``[1, B]``),
        returns logits ``[B, V]`` (schedule_infer.py:409-449).  ``position`` is checked against each
        sequence's own length when given (an int, or one value per sequence)."""
        tok = input_token.reshape(-1)
        B = len(self._batch)
        if tok.numel() != B:
            raise ValueError(f"decode_step needs one token per sequence: got {tok.numel()} for batch {B}")
        if position is not None:
            want = [int(position)] * B if not hasattr(position, "__len__") else [int(p) for p in position]
            have = [self.planner.context_len(b) for b in self._batch]
            if want != have:
                raise ValueError(f"position {want} does not match the cached lengths {have}")
        toks = {}
        for i, b in enumerate(self._batch):
            self._offset[b] = self.planner.context_len(b)
            toks[b] = tok[i:i + 1]
        got = self._step(toks)
        if len(got) != B:
            raise RuntimeError("not every sequence could be scheduled in this decode step")
        return torch.stack([got[b] for b in self._batch])

    def fork(self, row: int) -> int:
        """A second sequence with the tokens of batch row ``row`` so far (several continuations of one prompt): the new batch
        row, the last one.  Its full blocks are shared, its last block is copied in every layer's pools."""
        new = max(self._batch) + 1
        self.backend.copy_blocks(self.planner.fork(self._batch[row], new))
        self._batch.append(new)
        self._offset[new] = self._offset.get(self._batch[row], 0)
        return len(self._batch) - 1

    def clear_cache(self) -> None:
        """Release every sequence of the current batch (schedule_infer.py:451-454)."""
        for b in self._batch:
            try:
                self.planner.finish(b)
            except ValueError:
                pass
        self._batch = []
