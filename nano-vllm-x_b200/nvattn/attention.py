"""Drop-in replacement for ``nanovllm.layers.attention.Attention``.

Constructor, attributes and ``forward(q, k, v)`` follow
nanovllm/layers/attention.py:43-75 exactly:

* ``k_cache``/``v_cache`` start as empty tensors and are rebound by
  ``ModelRunner.allocate_kv_cache`` (model_runner.py:117-121), which finds
  the module through ``hasattr(module, "k_cache")``;
* ``forward`` reads only the attention context: it scatters the new K/V into
  the cache when one is bound (attention.py:61-63), then runs varlen prefill
  — over the caches when ``block_tables`` is set, i.e. a prefix-cache hit
  (attention.py:64-70) — or paged decode (attention.py:71-74);
* outputs have the reference's shapes: (N, H, d) for prefill and
  (B, 1, H, d) for decode.

``forward_fused`` is the same step with the producer side folded in: it
takes the raw q/k/v split of the QKV projection plus the RMSNorm weights and
the rotary cache, and one kernel applies q_norm/k_norm and the rotation and
scatters K/V (qwen3.py:82-86 and attention.py:62-63) before the attention.

The cache may also be bound as ``float8_e4m3fn`` pages with their exponent
bytes in ``k_scale``/``v_scale`` (``ops.store_kvcache_fp8``): new rows are then
quantised as they are scattered, decode attends the fp8 pages, and a
prefix-cache prefill reads its sequences back as dense bf16 rows first, a group
of sequences at a time so that these rows stay within about ``READ_BACK_KEYS``.

All steps run libnvattn kernels; there is no other code path.
"""
from __future__ import annotations

import torch
from torch import nn

from . import context as _ctx
from . import ops


# Keys per group of sequences that a prefill over an fp8 cache reads back (1 GB
# for 8 KV heads; one sequence may be longer)
READ_BACK_KEYS = 1 << 18


class Attention(nn.Module):
    # Source of the per-step context; ``nvattn.install`` points this at the
    # host engine's context module so both read the same global.
    get_context = staticmethod(_ctx.get_context)

    def __init__(self, num_heads, head_dim, scale, num_kv_heads):
        super().__init__()
        self.num_heads = num_heads
        self.head_dim = head_dim
        self.scale = scale
        self.num_kv_heads = num_kv_heads
        self.k_cache = self.v_cache = torch.tensor([])
        self.k_scale = self.v_scale = None  # exponent bytes of an fp8 cache

    def forward(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor):
        context = self.get_context()
        k_cache, v_cache = self.k_cache, self.v_cache
        if k_cache.numel() and v_cache.numel():
            self._store(k, v, context.slot_mapping)
        return self._attend(context, q, k, v)

    def _fp8(self) -> bool:
        if self.k_cache.dtype != torch.float8_e4m3fn:
            return False
        if self.k_scale is None or self.v_scale is None:
            raise ValueError("an fp8 cache needs its exponent bytes in k_scale and v_scale")
        return True

    def _store(self, k, v, slot_mapping):
        if self._fp8():
            ops.store_kvcache_fp8(k, v, self.k_cache, self.v_cache, self.k_scale, self.v_scale,
                                  slot_mapping)
        else:
            ops.store_kvcache(k, v, self.k_cache, self.v_cache, slot_mapping)

    def forward_fused(self, positions: torch.Tensor, q: torch.Tensor, k: torch.Tensor,
                      v: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                      cos_sin_cache: torch.Tensor, eps: float):
        """q_norm/k_norm + rotary_emb + KV scatter in one kernel, then attention.

        q, k, v are the un-normalised split of the QKV projection
        (qwen3.py:79-81); the result equals ``forward`` applied to the
        normalised, rotated q and k (qwen3.py:82-86).
        """
        context = self.get_context()
        k_cache, v_cache = self.k_cache, self.v_cache
        bound = bool(k_cache.numel() and v_cache.numel())
        # the rotated K itself is read only by dense prefill; the other paths
        # read K back from the cache
        need_k = bool(context.is_prefill and context.block_tables is None)
        if bound and self._fp8():  # the kernel scatters bf16 rows: quantise its K after it
            q, k = ops.qk_norm_rope_store(positions, q, k, v, q_weight, k_weight, cos_sin_cache,
                                          eps)
            self._store(k, v, context.slot_mapping)
            return self._attend(context, q, k, v)
        q, k = ops.qk_norm_rope_store(positions, q, k, v, q_weight, k_weight, cos_sin_cache, eps,
                                      k_cache if bound else None, v_cache if bound else None,
                                      context.slot_mapping if bound else None, need_k=need_k)
        return self._attend(context, q, k, v)

    def _attend(self, context, q: torch.Tensor, k, v):
        k_cache, v_cache = self.k_cache, self.v_cache
        if context.is_prefill:
            if context.block_tables is not None:  # prefix cache
                if self._fp8():
                    return self._prefill_fp8(context, q)
                k, v = k_cache, v_cache
            o = ops.varlen_prefill(q, k, v, context.cu_seqlens_q, context.cu_seqlens_k,
                                   context.max_seqlen_q, context.max_seqlen_k,
                                   softmax_scale=self.scale, causal=True,
                                   block_table=context.block_tables)
        elif self._fp8():
            o = ops.paged_decode_fp8(q, k_cache, v_cache, self.k_scale, self.v_scale,
                                     context.context_lens, context.block_tables,
                                     softmax_scale=self.scale).unsqueeze(1)
        else:  # decode
            o = ops.paged_decode(q, k_cache, v_cache, context.context_lens,
                                 context.block_tables, softmax_scale=self.scale).unsqueeze(1)
        return o

    def _prefill_fp8(self, context, q: torch.Tensor) -> torch.Tensor:
        """Prefix-cache prefill over an fp8 cache: the sequences' rows read back, then dense.

        The rows' number is on the device only, so each group of sequences gets
        room for max_seqlen_k apiece: ragged batches would claim many times their
        keys if all were read back at once. (A sequence may have one key more than
        its table, so that its length is flagged.) Rows behind the keys are left as
        they are: the prefill takes nothing from them.
        """
        table, cu_q, cu_k = context.block_tables, context.cu_seqlens_q, context.cu_seqlens_k
        longest = max(1, min(context.max_seqlen_k, table.shape[1] * self.k_cache.shape[1] + 1))
        step = max(1, READ_BACK_KEYS // longest)
        o = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        k, v = q.new_empty((2, min(step, table.shape[0]) * longest, *self.k_cache.shape[2:])).unbind()
        for b in range(0, table.shape[0], step):
            rows = table[b:b + step]
            n = rows.shape[0] * longest
            ck = cu_k[b:b + step + 1]
            ck = ck - ck[0]
            ops.load_kvcache_fp8(self.k_cache, self.v_cache, self.k_scale, self.v_scale, ck, rows, n,
                                 k[:n], v[:n])
            ops.varlen_prefill(q, k[:n], v[:n], cu_q[b:b + step + 1], ck, context.max_seqlen_q,
                               context.max_seqlen_k, softmax_scale=self.scale, causal=True, out=o)
        return o
