"""Decoding with a key / value cache in 8 bits: ``time_propagate`` (reference
athena/models/speech_transformer.py:164-194) for the newest position only.

The reference -- and ``SpeechTransformer.time_propagate`` -- runs the decoder over the whole history at
every step and projects the encoder output to keys and values again for every layer, step and
hypothesis.  ``CachedPropagate`` projects the encoder output once per utterance, keeps the keys and
values of the history, and computes one row per hypothesis and step.  All layers share the block tables
and lengths of a hypothesis; every hypothesis reads the same blocks of the encoder output.
"""
import math

import numpy as np
import torch

from .. import ops
from ..layers.attention import AttnMask
from ..layers.fused import LN_EPS, ffn_fwd, lin_fwd, lin_fwd_group

BLOCK = 16          # tokens of a block: label histories are some dozens long, and a beam copies whole blocks


class LayerCaches:
    """The 8-bit caches of all layers over one pool of blocks (see ``athena_kv8_append`` for the layout)."""

    def __init__(self, layers, blocks, heads, head_size, device):
        w = ops.kv8_width(head_size)
        self.k_codes = torch.zeros((layers, blocks, heads, BLOCK, w), dtype=torch.int8, device=device)
        self.v_codes = torch.zeros((layers, blocks, heads, w, BLOCK), dtype=torch.int8, device=device)
        self.k_scale = torch.zeros((layers, blocks, heads), dtype=torch.float32, device=device)
        self.v_scale = torch.zeros((layers, blocks, heads), dtype=torch.float32, device=device)

    def of(self, layer):
        return self.k_codes[layer], self.v_codes[layer], self.k_scale[layer], self.v_scale[layer]

    def copy_blocks(self, source):
        """The contents of the blocks ``source`` (int64), for ``paste``."""
        return [t.index_select(1, source) for t in (self.k_codes, self.v_codes, self.k_scale, self.v_scale)]

    def paste(self, target, contents):
        for t, c in zip((self.k_codes, self.v_codes, self.k_scale, self.v_scale), contents):
            t.index_copy_(1, target, c)


class CachedPropagate:
    """``time_propagate`` of a model for at most ``beam_size`` hypotheses at a time.  ``begin`` takes the encoder
    output of an utterance; each call then takes the hypotheses so far, like ``time_propagate``.  A hypothesis
    that extends one of the call before costs one row; anything else is computed afresh."""

    def __init__(self, model, beam_size):
        self.model = getattr(model, "model", model)         # MtlTransformerCtc holds a SpeechTransformer
        self.layers = list(self.model.transformer.decoder.layers)
        attn = self.layers[0].attn1
        self.heads, self.depth, self.d_model = attn.num_heads, attn.depth, attn.d_model
        ops.kv8_width(self.depth)
        if beam_size < 1:
            raise ValueError("CachedPropagate: beam_size %d" % beam_size)
        self.beam_size = int(beam_size)
        self.room = 0
        self.memory_frames = 0
        self.previous = None                                # the hypotheses of the call before, on the host

    def _make_room(self, labels):
        dev, width = self.model.store.device, -(-labels // BLOCK)
        self.room = width * BLOCK
        pool = self.beam_size * width
        self.cache = LayerCaches(len(self.layers), pool, self.heads, self.depth, dev)
        self.tables = torch.full((self.beam_size, width), -1, dtype=torch.int32, device=dev)
        self.free_blocks = torch.arange(pool, dtype=torch.int32, device=dev)
        self.free_count = torch.tensor([pool], dtype=torch.int32, device=dev)
        self.lens = torch.zeros(self.beam_size, dtype=torch.int32, device=dev)
        self.done = torch.full((self.beam_size,), -1, dtype=torch.int32, device=dev)
        self.previous = None

    def begin(self, encoder_output, memory_mask=None, max_labels=None):
        """Projects the encoder output [1, T', d] for all layers and forgets the hypotheses of the last utterance."""
        T, d = encoder_output.shape[1], encoder_output.shape[2]
        labels = T if max_labels is None else int(max_labels)
        dev = self.model.store.device
        self.model.store.refresh_shadows()
        if labels > self.room:
            self._make_room(labels)
        if T > self.memory_frames:
            self.memory_frames = -(-T // BLOCK) * BLOCK
            self.memory = LayerCaches(len(self.layers), self.memory_frames // BLOCK, self.heads, self.depth, dev)
            self.memory_table = torch.arange(self.memory_frames // BLOCK, dtype=torch.int32, device=dev)[None]
            self.memory_slots = torch.arange(self.memory_frames, dtype=torch.int32, device=dev)
        mask = AttnMask.coerce(memory_mask).key_mask
        with torch.no_grad():
            m2 = encoder_output[:1].contiguous().view(T, d)
            outs = lin_fwd_group([(m2, T, w) for l in self.layers for w in (l.attn2.wk, l.attn2.wv)])
            for i in range(len(self.layers)):
                ops.kv8_append(self._split(outs[2 * i]), self._split(outs[2 * i + 1]), self.memory_slots[:T], *self.memory.of(i))
            # (the input mask hides the frames behind an utterance's end)
            seen = torch.full((1,), T, dtype=torch.int32, device=dev) if mask is None else \
                (mask[:1] == 0).sum(dim=1, dtype=torch.int32)
            self.memory_lens = seen.expand(self.beam_size).contiguous()
        self.previous = None

    def _split(self, x):
        return x.view(x.shape[0], self.heads, self.depth)

    def _plan(self, n, new_rows, rows):
        return ops.kv_plan(self.lens[:n], new_rows, self.tables[:n], self.free_blocks, self.free_count, BLOCK, rows)

    def _rearrange(self, parents, length):
        """Row i goes on from what row parents[i] holds (``length`` tokens each)."""
        n, blocks = len(parents), -(-length // BLOCK)
        dev = self.lens.device
        source = self.tables[torch.tensor(parents, device=dev), :blocks].reshape(-1).long()
        contents = self.cache.copy_blocks(source)
        self._plan(self.beam_size, self.done, 0)
        self._plan(n, torch.full((n,), length, dtype=torch.int32, device=dev), n * length)
        self.cache.paste(self.tables[:n, :blocks].reshape(-1).long(), contents)

    def _parents(self, seqs):
        """For every hypothesis the row of the call before that it extends by one label, or None."""
        if self.previous is None or self.previous.shape[1] + 1 != seqs.shape[1]:
            return None
        rows = {tuple(r): i for i, r in reversed(list(enumerate(self.previous.tolist())))}
        parents = [rows.get(tuple(r)) for r in seqs[:, :-1].tolist()]
        return None if any(p is None for p in parents) else parents

    def __call__(self, history_logits, history_predictions, step, enc_outputs=None):
        """Logits [n, num_class] of the newest position, as ``time_propagate`` returns them."""
        if isinstance(history_predictions, (list, tuple)):
            history_predictions = torch.stack([torch.as_tensor(t) for t in history_predictions], dim=1)
        seqs = np.asarray(torch.as_tensor(history_predictions).cpu(), dtype=np.int64)
        n, length = seqs.shape
        if not 1 <= n <= self.beam_size or self.memory_frames == 0:
            raise RuntimeError("CachedPropagate: %d hypotheses, made for 1 to %d, after begin()" % (n, self.beam_size))
        if length > self.room:
            raise RuntimeError("CachedPropagate: histories of %d labels, begin() made room for %d" % (length, self.room))
        dev = self.lens.device
        with torch.no_grad():
            self.model.store.refresh_shadows()
            parents = self._parents(seqs)
            if parents is None:                             # from the beginning
                self._plan(self.beam_size, self.done, 0)
                fresh, first = length, 0
            else:
                if parents != list(range(self.previous.shape[0])):
                    self._rearrange(parents, length - 1)
                fresh, first = 1, length - 1
            plan = self._plan(n, torch.full((n,), fresh, dtype=torch.int32, device=dev), n * fresh)
            y = self._decoder(torch.as_tensor(seqs[:, first:], device=dev).to(torch.int32).contiguous(), plan, n, fresh, first)
            last = y.view(n, fresh, self.d_model)[:, -1:].contiguous()
            logits = self.model._project(self.model.final_layer, last)[:, -1, :].to(torch.float32)
        self.previous = seqs.copy()
        return logits, list(history_logits) + [logits], step + 1

    def _decoder(self, ids, plan, n, fresh, first):
        """The decoder stack on the new rows ``ids`` [n, fresh], the first of them at position ``first``."""
        net, M = self.model.y_net, n * fresh
        st = net.store
        x = torch.empty((M, self.d_model), dtype=st.compute_dtype, device=ids.device)
        ops.embed_fwd(net.embedding, ids, st.pe(self.d_model)[first:], n, fresh, self.d_model, net.num_class, net.xscale, 0.0,
                      st.rng_state, net.site_drop, x)
        scale = 1.0 / math.sqrt(self.depth)
        cu = plan.cu_rows if fresh > 1 else None
        table = self.memory_table.expand(n, -1)
        x32 = None
        for i, layer in enumerate(self.layers):
            q, k, v = lin_fwd_group([(x, M, w) for w in (layer.attn1.wq, layer.attn1.wk, layer.attn1.wv)])
            ops.kv8_append(self._split(k), self._split(v), plan.slots, *self.cache.of(i))
            a = ops.kv8_attention(self._split(q), *self.cache.of(i), self.tables[:n], self.lens[:n], cu_rows=cu, max_rows=fresh,
                                  causal=True, scale=scale)
            x, x32 = self._normed(x, x32, lin_fwd(a.view(M, -1), M, layer.attn1.dense)[0], layer.norm1)
            q, _ = lin_fwd(x, M, layer.attn2.wq)
            a = ops.kv8_attention(self._split(q), *self.memory.of(i), table, self.memory_lens[:n], cu_rows=cu, max_rows=fresh,
                                  causal=False, scale=scale)
            x, x32 = self._normed(x, x32, lin_fwd(a.view(M, -1), M, layer.attn2.dense)[0], layer.norm2)
            f, _ = ffn_fwd(x, M, layer, 0.0, st.rng_state)
            x, x32 = self._normed(x, x32, f, layer.norm3)
        return x

    def _normed(self, x, x32, a, norm):
        """LayerNorm(x + a); where the kernels cover the width the residual stream passes on in fp32."""
        wide = ops.layernorm_wide_ok(a) and x.is_contiguous()
        r = ops.add_layernorm_fwd(x, a, norm.gamma, norm.beta, LN_EPS, 0.0, self.model.store.rng_state, 0,
                                  a32=x32 if wide else None, want_y32=wide)
        return r[1], (r[4] if wide else None)


class LogitRules:
    """Penalties, biases and a grammar for the classes of a beam search (``ops.logits_process``).

    ``repetition`` (> 1 makes labels of the hypothesis less likely), ``presence``, ``frequency``: see
    ``athena_logits_process``; ``bias``: {class: value}; ``grammar``: a callable that takes the hypotheses
    [n, length] (numpy, <sos> first) and returns a bool array [n, num_class], the classes each may go on with."""

    def __init__(self, repetition=1.0, presence=0.0, frequency=0.0, bias=None, grammar=None):
        if repetition <= 0:
            raise ValueError("LogitRules: repetition must be positive")
        self.repetition, self.presence, self.frequency = float(repetition), float(presence), float(frequency)
        self.bias = {int(k): float(v) for k, v in (bias or {}).items()}
        self.grammar = grammar

    def __bool__(self):
        return self.repetition != 1.0 or self.presence != 0.0 or self.frequency != 0.0 or bool(self.bias) or self.grammar is not None

    def __call__(self, logits, seqs):
        """Logits [n, num_class] on the GPU of the hypotheses ``seqs`` [n, length]; <sos> does not count as a label."""
        n, V = logits.shape
        dev = logits.device
        kw = {}
        if self.repetition != 1.0 or self.presence != 0.0 or self.frequency != 0.0:
            full = lambda v: torch.full((n,), v, dtype=torch.float32, device=dev)
            kw = dict(history=torch.as_tensor(np.ascontiguousarray(seqs[:, 1:], dtype=np.int32), device=dev), repetition=full(self.repetition),
                      presence=full(self.presence), frequency=full(self.frequency))
        if self.bias:
            kw.update(bias_ids=torch.tensor(list(self.bias), dtype=torch.int32, device=dev),
                      bias_values=torch.tensor(list(self.bias.values()), dtype=torch.float32, device=dev))
        if self.grammar is not None:
            kw["allowed"] = pack_classes(self.grammar(seqs)).to(dev)
        return ops.logits_process(logits, **kw)


def pack_classes(allowed):
    """A bool array [n, classes] as the bit mask of ``ops.logits_process``: int32 [n, ceil(classes / 32)]."""
    bits = np.asarray(allowed, dtype=bool)
    if bits.ndim != 2:
        raise ValueError("pack_classes: [n, classes] expected")
    words = -(-bits.shape[1] // 32)
    padded = np.zeros((bits.shape[0], words * 32), dtype=bool)
    padded[:, :bits.shape[1]] = bits
    return torch.from_numpy(np.packbits(padded, axis=1, bitorder="little").view("<i4").astype(np.int32))
