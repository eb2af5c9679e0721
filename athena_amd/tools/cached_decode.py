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
    that extends one of the call before costs one row; anything else is computed afresh.

    Such a step is some thirty small launches whose shapes depend on the number of hypotheses alone (positions,
    lengths and tables live on the GPU), so it is recorded into a HIP graph the second time a number comes up
    (``graph`` false: never).  One stream at a time: like every layer, the projections share the library's
    workspace of the device."""

    def __init__(self, model, beam_size, graph=True):
        self.model = getattr(model, "model", model)         # MtlTransformerCtc holds a SpeechTransformer
        self.layers = list(self.model.transformer.decoder.layers)
        attn = self.layers[0].attn1
        self.heads, self.depth, self.d_model = attn.num_heads, attn.depth, attn.d_model
        ops.kv8_width(self.depth)
        if beam_size < 1:
            raise ValueError("CachedPropagate: beam_size %d" % beam_size)
        self.beam_size, self.graph = int(beam_size), bool(graph)
        self.room = 0
        self.memory_frames = 0
        self.previous = None                                # the hypotheses of the call before, on the host
        self.recorded = {}                                  # hypotheses -> (graph, logits); 0 after one eager step

    def _make_room(self, labels):
        # (at least twice the room before, here and for the memory: what is recorded holds these tensors, and a row of ever longer
        # utterances would make new ones and record every step again for each of them: recording alone 0.7 ms a step of 40, replays 0.56)
        dev, width = self.model.store.device, max(-(-labels // BLOCK), 2 * self.room // BLOCK)
        self.room = width * BLOCK
        pool = self.beam_size * width
        # (one block more than there are to give: what a copy of unused table entries goes to)
        self.cache = LayerCaches(len(self.layers), pool + 1, self.heads, self.depth, dev)
        self.spare = pool
        self.tables = torch.full((self.beam_size, width), -1, dtype=torch.int32, device=dev)
        self.free_blocks = torch.arange(pool, dtype=torch.int32, device=dev)
        self.free_count = torch.tensor([pool], dtype=torch.int32, device=dev)
        self.lens = torch.zeros(self.beam_size, dtype=torch.int32, device=dev)
        self.done = torch.full((self.beam_size,), -1, dtype=torch.int32, device=dev)
        self.one = torch.ones(self.beam_size, dtype=torch.int32, device=dev)
        self.ids = torch.zeros(self.beam_size, dtype=torch.int32, device=dev)
        self.parents = torch.zeros(self.beam_size, dtype=torch.int64, device=dev)
        self.previous = None
        self._forget_recorded()

    def _forget_recorded(self):
        if any(self.recorded.values()):
            torch.cuda.synchronize()                        # (the last replay may still be under way)
        self.recorded = {}

    def begin(self, encoder_output, memory_mask=None, max_labels=None):
        """Projects the encoder output [1, T', d] for all layers and forgets the hypotheses of the last utterance.
        ``memory_mask`` hides frames behind the utterance's end only: the cache knows a length, no holes."""
        T, d = encoder_output.shape[1], encoder_output.shape[2]
        mask, frames = AttnMask.coerce(memory_mask).key_mask, T
        if mask is not None:
            hidden = mask[0].cpu().numpy() != 0
            frames = int((~hidden).sum())
            if hidden.shape[0] != T or frames == 0 or hidden[:frames].any():
                raise RuntimeError("CachedPropagate: the memory mask must leave the first of %d frames and hide the others" % T)
        labels = T if max_labels is None else int(max_labels)
        dev = self.model.store.device
        self.model.store.refresh_shadows()
        if labels > self.room:
            self._make_room(labels)
        if T > self.memory_frames:
            self.memory_frames = max(-(-T // BLOCK) * BLOCK, 2 * self.memory_frames)
            self.memory = LayerCaches(len(self.layers), self.memory_frames // BLOCK, self.heads, self.depth, dev)
            self.memory_table = torch.arange(self.memory_frames // BLOCK, dtype=torch.int32, device=dev)[None]
            self.memory_slots = torch.arange(self.memory_frames, dtype=torch.int32, device=dev)
            self.memory_lens = torch.zeros(self.beam_size, dtype=torch.int32, device=dev)
            self._forget_recorded()
        with torch.no_grad():
            m2 = encoder_output[:1].contiguous().view(T, d)
            outs = lin_fwd_group([(m2, T, w) for l in self.layers for w in (l.attn2.wk, l.attn2.wv)])
            for i in range(len(self.layers)):
                ops.kv8_append(self._split(outs[2 * i]), self._split(outs[2 * i + 1]), self.memory_slots[:T], *self.memory.of(i))
            self.memory_lens.fill_(frames)
        self.previous = None

    def _split(self, x):
        return x.view(x.shape[0], self.heads, self.depth)

    def _plan(self, n, new_rows, rows):
        return ops.kv_plan(self.lens[:n], new_rows, self.tables[:n], self.free_blocks, self.free_count, BLOCK, rows)

    def _rearrange(self, n):
        """Row i goes on from what row ``parents[i]`` holds: everything is copied aside, all blocks are given back, and
        the contents go into the blocks of a new plan."""
        parents = self.parents[:n]
        lens = self.lens.index_select(0, parents)
        spare = lambda table: torch.where(table < 0, self.spare, table).reshape(-1).long()
        contents = self.cache.copy_blocks(spare(self.tables.index_select(0, parents)))
        self._plan(self.beam_size, self.done, 0)
        self.tables.fill_(-1)
        self._plan(n, lens, n * self.room)
        self.cache.paste(spare(self.tables[:n]), contents)

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
        positions = self.model.store.pe(self.d_model).shape[0]
        # (labels that there are not are taken for the nearest one, as time_propagate does)
        labels = np.clip(seqs, 0, self.model.y_net.num_class - 1).astype(np.int32)
        if length > min(self.room, positions):
            raise RuntimeError("CachedPropagate: histories of %d labels, begin() made room for %d, the positional table for %d"
                               % (length, self.room, positions))
        with torch.no_grad():
            self.model.store.refresh_shadows()
            parents, self.previous = self._parents(seqs), None      # (a step that fails leaves no half history behind)
            if parents is None:                             # from the beginning
                self._plan(self.beam_size, self.done, 0)
                self.tables.fill_(-1)
                ids = torch.from_numpy(np.ascontiguousarray(labels)).to(self.lens.device)
                logits = self._rows(ids.view(-1), n, length, torch.full((n,), length, dtype=torch.int32, device=self.lens.device))
            else:
                self.ids[:n].copy_(torch.from_numpy(np.ascontiguousarray(labels[:, -1])))
                self.parents[:n].copy_(torch.tensor(parents, dtype=torch.int64))
                logits = self._step(n)
        self.previous = seqs.copy()
        return logits, list(history_logits) + [logits], step + 1

    def _step(self, n):
        """One row for each of ``n`` hypotheses, from ``ids`` and ``parents``: eagerly the first time, then replayed."""
        kept = self.recorded.get(n)
        if kept is None:
            self.recorded[n] = 0
            return self._extend(n)
        if kept == 0:
            if not self.graph or torch.cuda.is_current_stream_capturing():
                return self._extend(n)
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            graph = torch.cuda.CUDAGraph()
            # (other host threads, a data loader's say, may go on with calls of their own meanwhile)
            with torch.cuda.graph(graph, stream=side, capture_error_mode="thread_local"):
                logits = self._extend(n)
            kept = self.recorded[n] = (graph, logits)
        kept[0].replay()
        return kept[1].clone()                              # (the next replay writes there again)

    def _extend(self, n):
        self._rearrange(n)
        return self._rows(self.ids[:n], n, 1, self.one[:n])

    def _rows(self, ids, n, fresh, new_rows):
        """Logits [n, num_class] of the last of ``fresh`` new rows of every hypothesis."""
        plan = self._plan(n, new_rows, n * fresh)
        net, M = self.model.y_net, n * fresh
        st = net.store
        # embedding * sqrt(d) + positional table, each row at its own position
        x = net.embedding.index_select(0, ids.long()).mul_(net.xscale).add_(st.pe(self.d_model).index_select(0, plan.positions.long()))
        x = x.to(st.compute_dtype)
        scale, cu = 1.0 / math.sqrt(self.depth), plan.cu_rows if fresh > 1 else None
        table = self.memory_table.expand(n, -1)
        x32 = qkv = None
        for i, layer in enumerate(self.layers):
            nxt = self.layers[i + 1] if i + 1 < len(self.layers) else None
            q, k, v = qkv if qkv is not None else lin_fwd_group([(x, M, w) for w in (layer.attn1.wq, layer.attn1.wk, layer.attn1.wv)])
            ops.kv8_append(self._split(k), self._split(v), plan.slots, *self.cache.of(i))
            a = ops.kv8_attention(self._split(q), *self.cache.of(i), self.tables[:n], self.lens[:n], cu_rows=cu, max_rows=fresh,
                                  causal=True, scale=scale).view(M, self.d_model)
            tail = ops.layer_tail_ok(x, self.d_model, layer.attn1.dense) and \
                ops.layer_tail_ok(x, self.d_model, layer.attn2.dense, layer.ffn0, layer.ffn1)
            cross = lambda q: ops.kv8_attention(self._split(q), *self.memory.of(i), table, self.memory_lens[:n], cu_rows=cu,
                                                max_rows=fresh, causal=False, scale=scale).view(M, self.d_model)
            if tail:
                # projection, residual and LayerNorm in one launch each, the next projections with them (see
                # DecoderLayerFn); the residual stream passes on in fp32
                t = ops.layer_tail_fwd(a, x, layer.attn1.dense, layer.norm1, None, None, None, LN_EPS, 0.0, st.rng_state, 0, 0, 0,
                                       next_qkv=(layer.attn2.wq,), x32=x32, want_y32=True)
                b = ops.layer_tail_fwd(cross(t["q"]), t["y1"], layer.attn2.dense, layer.norm2, layer.ffn0, layer.ffn1, layer.norm3,
                                       LN_EPS, 0.0, st.rng_state, 0, 0, 0,
                                       next_qkv=(nxt.attn1.wq, nxt.attn1.wk, nxt.attn1.wv) if nxt is not None else None,
                                       x32=t["y32"], want_y32=True)
                x, x32 = b["y2"], b["y32"]
                qkv = (b["q"], b["k"], b["v"]) if nxt is not None else None
                continue
            x, x32 = self._normed(x, x32, lin_fwd(a, M, layer.attn1.dense)[0], layer.norm1)
            x, x32 = self._normed(x, x32, lin_fwd(cross(lin_fwd(x, M, layer.attn2.wq)[0]), M, layer.attn2.dense)[0], layer.norm2)
            x, x32 = self._normed(x, x32, ffn_fwd(x, M, layer, 0.0, st.rng_state)[0], layer.norm3)
            qkv = None
        last = x.view(n, fresh, self.d_model)[:, -1:].contiguous()
        return self.model._project(self.model.final_layer, last)[:, -1, :].to(torch.float32)

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
    [n, length] (numpy, <sos> first) and returns a bool array [n, num_class], the classes each may go on with.  It is
    asked about hypotheses that it allowed itself only; where none of them ends in time the search raises RuntimeError."""

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
