"""Loop restatements, in whole numbers and 64 bits on the CPU, of the decoding operators: block plans, the
8-bit key/value cache, attention over it, penalties and masks on logits."""
import math

import torch


def plan(lens, new_rows, tables, free_blocks, free_count, block_size, rows):
    """What ``athena_kv_plan`` leaves: a dict of Python lists (cu_rows, slots, positions, lens, free_count, tables,
    free_blocks, status).  ``tables`` is a list of lists, ``free_blocks`` a list."""
    B, width = len(lens), len(tables[0])
    tables, free = [list(r) for r in tables], list(free_blocks)
    blocks = lambda n: -(-n // block_size)
    bad = [n < 0 or n + max(r, 0) > width * block_size for n, r in zip(lens, new_rows)]
    good = [(n, r) for n, r, x in zip(lens, new_rows, bad) if not x]
    taken = sum(blocks(n + r) - blocks(n) for n, r in good if r >= 0)
    given = sum(blocks(n) for n, r in good if r < 0)
    total = sum(r for _, r in good if r >= 0)
    level = free_count + given
    status = [max(taken - level, 0), sum(bad), max(total - rows, 0), max(level - len(free), 0)]
    if any(status):
        return dict(cu_rows=[0] * (B + 1), slots=[-1] * rows, positions=[0] * rows, lens=list(lens), free_count=free_count,
                    tables=tables, free_blocks=free, status=status)
    count = free_count
    for b in range(B):
        if new_rows[b] < 0:
            for j in range(blocks(lens[b])):
                free[count] = tables[b][j]
                count += 1
    cu, slots, positions, out = [0], [], [], []
    for b in range(B):
        r = max(new_rows[b], 0)
        for j in range(blocks(lens[b]), blocks(lens[b] + r) if new_rows[b] >= 0 else 0):
            count -= 1
            tables[b][j] = free[count]
        for p in range(lens[b], lens[b] + r):
            block = tables[b][p // block_size]
            slots.append(block * block_size + p % block_size if block >= 0 else -1)
            positions.append(p)
        cu.append(cu[-1] + r)
        out.append(lens[b] + r if new_rows[b] >= 0 else 0)
    pad = rows - len(slots)
    return dict(cu_rows=cu, slots=slots + [-1] * pad, positions=positions + [0] * pad, lens=out, free_count=count,
                tables=tables, free_blocks=free, status=status)


def append(x, slots, codes, scale):
    """``x`` [rows, heads, dk] into ``codes`` int8 [blocks, heads, block_size, width] and ``scale`` fp32 [blocks, heads], in
    place (``v_codes`` are passed with their last two axes exchanged)."""
    nb, heads, bs, width = codes.shape
    dk = x.shape[2]
    runs = []                                               # (block, rows): skipped rows do not end a run
    for t, s in enumerate(slots):
        if 0 <= s < nb * bs:
            if runs and runs[-1][0] == s // bs:
                runs[-1][1].append(t)
            else:
                runs.append((s // bs, [t]))
    for block, mine in runs:
        places = [slots[t] % bs for t in mine]
        first = min(places)
        for h in range(heads):
            rows = x[mine, h].double()
            top = (rows.abs().max() / 127).float()          # (NaN where a value is)
            old = scale[block, h] if first else torch.zeros(())
            if not torch.isfinite(top) or not torch.isfinite(old):
                scale[block, h] = float("nan")              # (infinity or NaN: the block stands for NaN either way)
                continue
            new = torch.maximum(old, top)
            if new > old:
                codes[block, h, :first] = torch.round(codes[block, h, :first].double() * old.double() / new.double()).to(torch.int8)
            for p, row in zip(places, rows):
                codes[block, h, p] = 0
                if new > 0:
                    codes[block, h, p, :dk] = torch.round(row / new.double()).clamp(-127, 127).to(torch.int8)
            scale[block, h] = new


def attention(q, k_codes, v_codes, k_scale, v_scale, tables, lens, cu_rows, causal, scale):
    """(out, lse, spread) in 64 bits; ``spread`` [rows, heads, dk] = sum_j p_j |v_j|, what relative errors of the
    probabilities act on.  Rows of no sequence stay NaN."""
    n, h, dk = q.shape
    nb, hk, bs, width = k_codes.shape
    out = torch.full((n, h, dk), math.nan, dtype=torch.float64)
    lse, spread = torch.full((n, h), math.nan, dtype=torch.float64), torch.full((n, h, dk), math.nan, dtype=torch.float64)
    for b in range(len(lens)):
        length = min(max(lens[b], 0), tables.shape[1] * bs)
        held = [j for j in range(length) if 0 <= int(tables[b, j // bs]) < nb]
        lo, hi = (max(cu_rows[b], 0), min(cu_rows[b + 1], n)) if cu_rows is not None else (b, b + 1)
        if hi <= lo:
            continue
        at = torch.tensor([int(tables[b, j // bs]) for j in held], dtype=torch.long)
        place = torch.tensor([j % bs for j in held], dtype=torch.long)
        for g in range(hk):
            k = (k_codes[at, g, place, :dk].double() * k_scale[at, g].double()[:, None]) if held else torch.zeros(0, dk).double()
            v = (v_codes[at, g, :dk, place].double() * v_scale[at, g].double()[:, None]) if held else torch.zeros(0, dk).double()
            for i in range(g * (h // hk), (g + 1) * (h // hk)):
                for t in range(lo, hi):
                    last = length - (hi - t) if causal else length - 1
                    see = [m for m, j in enumerate(held) if j <= last]
                    if not see:
                        out[t, i], lse[t, i], spread[t, i] = 0.0, -math.inf, 0.0
                        continue
                    w = (k[see] @ q[t, i].double()) * scale
                    p = torch.softmax(w, 0)
                    out[t, i], lse[t, i], spread[t, i] = p @ v[see], torch.logsumexp(w, 0), p @ v[see].abs()
    return out, lse, spread


def logits(x, history=None, history_len=None, repetition=None, presence=None, frequency=None, bias=None, bias_ids=None,
           bias_values=None, allowed=None):
    x = x.double().clone()
    R, V = x.shape
    for r in range(R):
        if history is not None:
            count = {}
            for i in history[r, :int(history_len[r]) if history_len is not None else None].tolist():
                if 0 <= i < V:
                    count[i] = count.get(i, 0) + 1
            for v, c in count.items():
                if repetition is not None:
                    x[r, v] = x[r, v] / repetition[r].double() if x[r, v] > 0 else x[r, v] * repetition[r].double()
                x[r, v] -= (frequency[r].double() * c if frequency is not None else 0) + \
                    (presence[r].double() if presence is not None else 0)
        if bias is not None:
            x[r] += bias[r if bias.dim() == 2 and bias.shape[0] == R else 0].double() if bias.dim() == 2 else bias.double()
        if bias_ids is not None:
            ids, values = (t[r if t.dim() == 2 and t.shape[0] == R else 0] if t.dim() == 2 else t for t in (bias_ids, bias_values))
            for i, b in zip(ids.tolist(), values.tolist()):
                if 0 <= i < V:
                    x[r, i] += b
        if allowed is not None:
            words = (allowed[r if allowed.shape[0] == R else 0] if allowed.dim() == 2 else allowed).tolist()
            for v in range(V):
                if not (words[v // 32] >> (v % 32)) & 1:
                    x[r, v] = -math.inf
    return x
