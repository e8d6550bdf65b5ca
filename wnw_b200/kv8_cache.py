"""``KV8Cache``: the full context of every head, held in 8 bits.

A cache for the session beside ``B200WnWCache``: instead of offloading chunks
of some heads it keeps every token of every head on the GPU, in half the bytes
(``wnw_b200.kv8``): paged, 8-bit codes with a scale for each block of 32
tokens and head, the newest tokens of each head in the model's type.  It
implements the same hooks (src/common/kv/flat_cache.py:161-186), so
``WnWSession`` and ``model.generate(past_key_values=cache)`` drive it; it needs
no class-A scores and no config.

With an adapter that hands positions instead of cosine tables
(``wnw_b200.adapters.RotaryAdapter``) a decode step of a layer is two launches:
the append, which rotates the step's keys and queries on the way, and the
attention, which starts streaming the older blocks while the append finishes.
"""
from __future__ import annotations

import torch

from wnw_b200.flat_cache import FlatVarlenCache
from wnw_b200.kv8 import KV8Attention, KV8Store, check_group, check_layout


class KV8Cache(FlatVarlenCache):
    """Constructor arguments as ``FlatVarlenCache`` (head_dim 64 or 128, one to
    eight query heads a kv head, a model in bf16 or fp16); optional: ``code``
    ("e4m3" or "int8"), ``page_rows`` (tokens a page), ``max_decode_tokens``
    (pages reserved for decoding at prefill; more are added on demand, an eighth
    of the context at least)."""

    #: what the session asks a cache: does it rank audio tokens at prefill,
    #: and does it rotate a decode step's queries and keys itself
    needs_prefill_scores = False
    rotates_decode = True

    def __init__(self, num_layers, num_kv_heads, num_q_heads, head_dim, device, adapter=None, *, code="e4m3",
                 page_rows=128, max_decode_tokens=1024):
        check_layout(head_dim, page_rows, code)
        if num_kv_heads < 1 or num_q_heads % num_kv_heads:
            raise ValueError(f"{num_q_heads} query heads over {num_kv_heads} kv heads: a multiple of them")
        check_group(num_q_heads // num_kv_heads)
        super().__init__(num_layers, num_kv_heads, num_q_heads, head_dim, device, adapter)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.code, self.page_rows, self.max_decode_tokens = code, page_rows, max(1, int(max_decode_tokens))
        self._clear()

    def _clear(self):
        self.stores = [None] * self.num_layers
        self._attention = [None] * self.num_layers
        self._new = [None] * self.num_layers
        self._rotation = None
        self._len = self._next = self._counts = self._starts = None
        self._prompt = self._room = self._step = 0
        self._prompt_rows = []  # per sample, without padding

    def setup_audio(self, audio_starts, audio_ends, attention_mask=None):
        super().setup_audio(audio_starts, audio_ends, attention_mask)
        self._clear()
        self.batch_size = int(audio_starts.shape[0])
        self._pads = self.pad_lens.tolist()

    def reset(self):
        super().reset()
        self._clear()

    # ------------------------------------------------------------- prefill
    def prefill_after_attn(self, layer_idx, class_a_scores, per_head_scores, key_states, value_states):
        """Append the prompt's keys and values (rotated by the model already),
        each sample from its first token that is not padding on."""
        B, H, S, D = key_states.shape
        if self._len is None:
            if B != self.batch_size:
                raise ValueError(f"a batch of {B} samples: setup_audio was given {self.batch_size}")
            self._starts = self.pad_lens.to(torch.int32)
            self._counts = S - self._starts
            self._len = torch.zeros(B * H, dtype=torch.int32, device=self.device)
            self._next = self._counts.repeat_interleave(H)
            self._prompt, self._prompt_rows = S, [S - p for p in self._pads]
            self._room = self._whole_pages(S + self.max_decode_tokens)
        pages = self._room // self.page_rows
        store = KV8Store(B * H, D, B * H * pages, pages, self.page_rows, self.code, key_states.dtype, self.device)
        store.reserve(self._room)
        store.append(key_states, value_states, self._len, starts=self._starts, counts=self._counts)
        self.stores[layer_idx] = store

    def prefill_all_layers_done(self):
        for s in self.stores:
            s.check()
        self._len.copy_(self._next)
        self._next = self._len + 1
        super().prefill_all_layers_done()
        self.stats.record_prefill(self._snapshot_cache_stats)

    # -------------------------------------------------------------- decode
    def decode_rotation(self, rotary, positions):
        """The coming layers' queries and keys arrive unrotated: rotate them by
        ``rotary`` at ``positions`` [axes, B, 1] on their way in (until the
        step's end)."""
        self._rotation = (rotary, positions)

    def decode_before_attn(self, layer_idx, k_new, v_new):
        if k_new.shape[-2] != 1:
            raise ValueError(f"a decode step of {k_new.shape[-2]} tokens: one at a time")
        if layer_idx == 0 and self._prompt + self._step + 1 > self._room:
            self._grow()
        self._new[layer_idx] = (k_new, v_new)
        store = self.stores[layer_idx]
        return store.pool, store.pool, self._next, self._prompt + self._step + 1

    def _whole_pages(self, rows):
        return -(-rows // self.page_rows) * self.page_rows

    def _grow(self):
        """Room for as many decode tokens again, in every layer, and an eighth
        more at least: each growth copies the layers' content."""
        self._room = self._whole_pages(self._room + max(self.max_decode_tokens, self._room // 8))
        for l, s in enumerate(self.stores):
            self.stores[l] = s.grown(self._room)
            self._attention[l] = None

    def fused_decode_attention(self, layer_idx, q_flat, q=None, k_flat=None, v_flat=None, cu_k=None, scale=None):
        """Append the step's token and attend: q_flat [segments, group, D]."""
        store, (k, v) = self.stores[layer_idx], self._new[layer_idx]
        B, H, G, D = self.batch_size, self.num_kv_heads, self.num_kv_groups, self.head_dim
        if self._rotation is None:
            store.append(k, v, self._len)
            q_flat = q_flat if q_flat.is_contiguous() else q_flat.contiguous()
        else:
            rotary, positions = self._rotation
            q_flat = store.append(k, v, self._len, rotary=rotary, positions=positions,
                                  q=q_flat.reshape(B, H * G, 1, D)).view(B * H, G, D)
        att = self._attention[layer_idx]
        if att is None or att.scale != float(scale):
            # layers run one after another on one stream: they share the first one's scratch
            first = next((a for a in self._attention if a is not None), None)
            att = self._attention[layer_idx] = KV8Attention(store, G, scale, scratch_of=first)
        # the append is the kernel right before: one token a segment is new
        return att(q_flat, self._next, fresh=1)

    def decode_all_layers_done(self):
        self._step += 1
        self._len.add_(1)
        self._next.add_(1)
        self._rotation = None
        if self.stats.enabled and self._step % self.stats.interval == 0:
            self.stats.record_decode(self._step, self._snapshot_cache_stats)

    def check(self):
        """Raise if a launch reported a problem on the device (a sync point)."""
        for s in self.stores:
            if s is not None:
                s.check()

    def layer_rows(self, layer_idx, seg):
        """(keys, values) fp32 of a segment as the cache reads back (between
        steps; for inspection)."""
        return self.stores[layer_idx].dequantize(seg, int(self._len[seg]))

    def _snapshot_cache_stats(self, step=-1):
        n = self.num_layers * self.num_kv_heads
        return [{"step": step, "gpu_total_tokens": n * (r + self._step)} for r in self._prompt_rows]
