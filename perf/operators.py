"""Cases and plain forms of the serving operators: block plans, the 8-bit key/value cache, attention over
it, and penalties, biases and grammar masks on logits.

``own`` false: elementary torch operations in 32 bits (64 where a value next to a rounding border
decides).  ``own`` true: the calls a decoding program makes of ``athena_amd.ops``.

The cache
  k_codes  int8 [blocks, kv_heads, block_size, width]   k_scale fp32 [blocks, kv_heads]
  v_codes  int8 [blocks, kv_heads, width, block_size]   v_scale fp32 [blocks, kv_heads]
An element stands for code * scale.  ``tables`` [sequences, table_width] int32 names the blocks of a sequence
in order; token t of a sequence lies in block tables[b, t // block_size] at t % block_size.
"""
import math

import torch

own = False


# ------------------------------------------------------------------------------------------ sizes
def _spread(low, high, n):
    """n whole numbers of [low, high], spread evenly and out of order, the same ones for every seed; the
    first is ``high``."""
    return [high - int((high - low + 1) * ((i * 0.6180339887498949) % 1.0)) for i in range(n)]


def _lens(case):
    if case.get("shared"):
        return [case["max_len"]] * case["batch"]
    return _spread(case["min_len"], case["max_len"], case["batch"])


def _rows(case, lens):
    """New rows of every sequence: at most its length."""
    if case["rows"] == 1:
        return [1] * case["batch"]
    return [min(n, r) for n, r in zip(lens, _spread(max(1, case["rows"] // 4), case["rows"], case["batch"]))]


def _width(head_size):
    return 32 if head_size <= 32 else 64 if head_size <= 64 else 128


def _visible(n, r, causal):
    """Query-key pairs of r new rows at the end of n tokens."""
    return r * n - (r * (r - 1) // 2 if causal else 0)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype).cuda()


_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------ cases
def listed():
    def attention(name, batch, heads, kv_heads, head_size, block, min_len, max_len, rows=1, causal=True, shared=False,
                  dtype="bf16"):
        return dict(name=name, op="attention", batch=batch, heads=heads, kv_heads=kv_heads, head_size=head_size, block=block,
                    min_len=min_len, max_len=max_len, rows=rows, causal=causal, shared=shared, dtype=dtype)

    return [
        # one step of a beam of ten label hypotheses: 4 heads of 64, a few dozen labels so far
        attention("attention_beam", 10, 4, 4, 64, 16, 7, 61),
        # the same beam's attention to the encoder output of one utterance (1000 frames, a quarter of them
        # after the front end): every hypothesis reads the same blocks; the fp32 precision mode
        attention("attention_memory", 10, 8, 8, 64, 16, 250, 250, causal=False, shared=True, dtype="fp32"),
        # a serving batch of ragged requests, grouped heads
        attention("attention_serve", 64, 32, 8, 128, 64, 60, 8192),
        # a few very long contexts: the split over the key axis
        attention("attention_long", 8, 32, 8, 128, 64, 120001, 131072),
        # chunks of prompts behind what is cached already
        attention("attention_chunk", 4, 32, 8, 128, 64, 2049, 16384, rows=512),
        # whole prompts, odd lengths, one head of queries per head of keys
        attention("attention_prompt", 3, 16, 16, 64, 32, 1501, 4001, rows=4001),
        # one new token per request, blocks partly filled
        dict(name="append_step", op="append", tokens=256, batch=256, kv_heads=8, head_size=128, block=64, dtype="bf16"),
        # chunks of prompts
        dict(name="append_chunk", op="append", tokens=8192, batch=16, kv_heads=8, head_size=128, block=64, dtype="bf16"),
        # a step of a small batch / a mixed batch of chunks and single tokens, some requests finished
        dict(name="plan_step", op="plan", batch=16, rows=1, block=16, table=64, finished=0),
        dict(name="plan_mixed", op="plan", batch=2048, rows=64, block=16, table=512, finished=50),
        # a beam of ten over the benchmark's vocabulary; a large batch over a large one
        dict(name="logits_beam", op="logits", rows=10, vocab=4233, history=61, biases=8, masked=True, dtype="fp32"),
        dict(name="logits_serve", op="logits", rows=256, vocab=131072, history=2000, biases=100, masked=True, dtype="bf16"),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "append", "plan", "logits"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op == "append":
        batch = _log_uniform(rng, 1, 256)
        return dict(op=op, tokens=max(batch, _log_uniform(rng, 1, 8192)), batch=batch, kv_heads=rng.choice([1, 2, 4, 8]),
                    head_size=rng.choice([8, 32, 64, 80, 128]), block=rng.choice([16, 32, 64, 128]), dtype=dtype)
    if op == "plan":
        return dict(op=op, batch=_log_uniform(rng, 1, 2048), rows=_log_uniform(rng, 1, 64), block=rng.choice([16, 32, 64]),
                    table=rng.choice([32, 100, 512]), finished=rng.choice([0, 1, 50]))
    if op == "logits":
        rows = _log_uniform(rng, 1, 256)
        return dict(op=op, rows=rows, vocab=_log_uniform(rng, 11, 131072), history=_log_uniform(rng, 1, 2000),
                    biases=rng.choice([0, 1, 100]), masked=rng.choice([True, False]), dtype=dtype)
    kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 7, 8])
    rows = rng.choice([1, 1, 1, 5, _log_uniform(rng, 2, 700)])
    top = 100000 if rows == 1 else 9000
    max_len = _log_uniform(rng, max(rows, 2), top)
    batch = min(_log_uniform(rng, 1, 128), max(1, 2 ** 20 // max_len), max(1, 2 ** 29 // (max_len * rows * kv_heads * group)))
    shared = rows == 1 and rng.random() < 0.2
    return dict(op=op, batch=batch, heads=kv_heads * group, kv_heads=kv_heads, head_size=rng.choice([8, 32, 64, 80, 128]),
                block=rng.choice([16, 32, 64, 128]), min_len=1 + max_len // rng.choice([2, 10, 100]), max_len=max_len,
                rows=rows, causal=rng.random() < 0.75, shared=shared, dtype=dtype)


# ------------------------------------------------------------------------------------------ inputs
def _prepare_attention(case, g):
    lens = _lens(case)
    rows = _rows(case, lens)
    block, hk, dk, width = case["block"], case["kv_heads"], case["head_size"], _width(case["head_size"])
    need = [-(-n // block) for n in lens]
    table_width = max(need) + 1
    blocks = (max(need) if case["shared"] else sum(need)) + 3
    order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    tables = torch.full((case["batch"], table_width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = order[at:at + n]
        at += 0 if case["shared"] else n
    # codes of normal values whose largest of a block lies about 3.5 deviations out; the deviations of
    # blocks and heads differ
    k_codes = torch.empty((blocks, hk, block, width), dtype=torch.int8, device="cuda")
    v_codes = torch.empty((blocks, hk, width, block), dtype=torch.int8, device="cuda")
    step = max(1, (1 << 27) // (hk * block * width))
    for i in range(0, blocks, step):
        for codes, cut in ((k_codes, (slice(None), slice(None), slice(None), slice(dk, None))),
                           (v_codes, (slice(None), slice(None), slice(dk, None), slice(None)))):
            part = torch.randn(codes[i:i + step].shape, generator=g, device="cuda").mul_(36.0).round_().clamp_(-127, 127)
            codes[i:i + step] = part.to(torch.int8)
            codes[i:i + step][cut] = 0                      # columns beyond the head size hold zeros
    spread = lambda: torch.exp(0.25 * torch.randn((blocks, hk), generator=g, device="cuda")) / 36.0
    k_scale, v_scale = spread(), spread()
    cu = [0]
    for r in rows:
        cu.append(cu[-1] + r)
    q = 1.5 * torch.randn((cu[-1], case["heads"], dk), generator=g, device="cuda")
    return dict(case=case, q=q.to(_TYPES[case["dtype"]]), k_codes=k_codes, v_codes=v_codes, k_scale=k_scale, v_scale=v_scale,
                tables=tables, lens=_ints(lens), cu_rows=None if max(rows) == 1 else _ints(cu), max_rows=max(rows),
                scale=1.0 / math.sqrt(dk))


def _append_layout(case):
    """(first token's place, number of tokens) of every sequence."""
    n = [case["tokens"] // case["batch"] + (i < case["tokens"] % case["batch"]) for i in range(case["batch"])]
    starts = _spread(0, case["block"] - 1, case["batch"])
    return list(zip(starts, n))


def _prepare_append(case, g):
    block, hk, dk, width = case["block"], case["kv_heads"], case["head_size"], _width(case["head_size"])
    layout = _append_layout(case)
    need = [-(-(s + n) // block) for s, n in layout]
    blocks = sum(need)
    order = torch.randperm(blocks, generator=g, device="cuda")
    # what the first block of a sequence holds already has about the size of what comes: some scales grow
    k_codes = torch.zeros((blocks, hk, block, width), dtype=torch.int8, device="cuda")
    v_codes = torch.zeros((blocks, hk, width, block), dtype=torch.int8, device="cuda")
    k_codes[..., :dk] = (torch.randn((blocks, hk, block, dk), generator=g, device="cuda") * 36).round().clamp(-127, 127).to(torch.int8)
    v_codes[:, :, :dk] = (torch.randn((blocks, hk, dk, block), generator=g, device="cuda") * 36).round().clamp(-127, 127).to(torch.int8)
    spread = lambda: torch.exp(0.1 * torch.randn((blocks, hk), generator=g, device="cuda")) / 36.0
    k_scale, v_scale = spread(), spread()
    slots, at = [], 0
    order_host = order.tolist()
    for (s, n), m in zip(layout, need):
        slots += [order_host[at + (s + i) // block] * block + (s + i) % block for i in range(n)]
        at += m
    t = _TYPES[case["dtype"]]
    k = torch.randn((case["tokens"], hk, dk), generator=g, device="cuda").to(t)
    v = torch.randn((case["tokens"], hk, dk), generator=g, device="cuda").to(t)
    return dict(case=case, k=k, v=v, slots=_ints(slots), k_codes=k_codes, v_codes=v_codes, k_scale=k_scale, v_scale=v_scale)


def _plan_sizes(case):
    """(lengths, new rows) of the requests: a third of them take a chunk, the others one row each, every
    few of them (one in 100 / ``finished``) are finished and give their blocks back (-1)."""
    top = case["table"] * case["block"] - case["rows"]
    lens = _spread(0, top, case["batch"])
    new = [r if i % 3 == 0 else 1 for i, r in enumerate(_spread(1, case["rows"], case["batch"]))]
    if case["finished"]:
        every = max(2, 100 // case["finished"])
        new = [-1 if i % every == 1 else r for i, r in enumerate(new)]
    return lens, new


def _prepare_plan(case, g):
    lens, new = _plan_sizes(case)
    block = case["block"]
    have = [-(-n // block) for n in lens]
    need = sum(-(-(n + r) // block) - h for n, r, h in zip(lens, new, have) if r > 0)
    pool = sum(have) + need + 17
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    column = torch.arange(case["table"], device="cuda")
    first = torch.tensor([0] + have[:-1], device="cuda").cumsum(0)
    held = torch.tensor(have, device="cuda")
    place = (first[:, None] + column[None]).clamp(max=pool - 1)
    tables = torch.where(column[None] < held[:, None], order[place], -1).to(torch.int32).contiguous()
    free = torch.full((pool,), -1, dtype=torch.int32, device="cuda")
    count = pool - sum(have)
    free[:count] = order[sum(have):]
    total = sum(max(r, 0) for r in new)
    return dict(case=case, lens=_ints(lens), new_rows=_ints(new), tables=tables, free_blocks=free, free_count=_ints([count]),
                rows=total + 5)                             # the batch is padded by five rows


def _prepare_logits(case, g):
    R, V, L = case["rows"], case["vocab"], case["history"]
    logits = 3.0 * torch.randn((R, V), generator=g, device="cuda")
    history = (torch.rand((R, L), generator=g, device="cuda").square() * V).to(torch.int32)     # low ids come often
    history_len = _ints(_spread(max(1, L // 4), L, R))
    even = lambda low, high: torch.rand(R, generator=g, device="cuda") * (high - low) + low
    state = dict(case=case, logits=logits.to(_TYPES[case["dtype"]]), history=history, history_len=history_len,
                 repetition=even(1.0, 1.5), presence=even(0.0, 0.5), frequency=even(0.0, 0.2), bias_ids=None,
                 bias_values=None, allowed=None)
    if case["biases"]:
        n = case["biases"]
        # ids differ within a row; a few entries are not in use
        ids = (torch.randint(0, V, (R, 1), generator=g, device="cuda") + torch.arange(n, device="cuda")[None] * (V // n if V >= n else 1)) % V
        ids = torch.where(torch.arange(n, device="cuda")[None] < min(n, V), ids, -1)
        state["bias_ids"] = torch.where(torch.rand((R, n), generator=g, device="cuda") < 0.9, ids, -1).to(torch.int32)
        state["bias_values"] = 2.0 * torch.randn((R, n), generator=g, device="cuda")
    if case["masked"]:
        # a grammar allows a quarter of the classes: one bit each, 32 to a word
        words = (V + 31) // 32
        a, b = (torch.randint(-2 ** 31, 2 ** 31, (R, words), generator=g, device="cuda", dtype=torch.int64) for _ in range(2))
        state["allowed"] = (a & b).to(torch.int32)
    return state


def prepare(case, seed):
    g = _generator(seed)
    return {"attention": _prepare_attention, "append": _prepare_append, "plan": _prepare_plan,
            "logits": _prepare_logits}[case["op"]](case, g)


# ------------------------------------------------------------------------------------------ plain forms
def _plain_attention(s):
    c = s["case"]
    q, lens = s["q"].float(), s["lens"].long()
    B, hk, dk, block = c["batch"], c["kv_heads"], c["head_size"], c["block"]
    group, R = c["heads"] // hk, s["max_rows"]
    cu = s["cu_rows"].long() if s["cu_rows"] is not None else torch.arange(B + 1, device=q.device)
    table = s["tables"].long().clamp(min=0)
    L = table.shape[1] * block
    # [B, kv_heads, L, dk] and [B, kv_heads, dk, L] in 32 bits
    k = (s["k_codes"][table][..., :dk] * s["k_scale"][table][..., None, None]).permute(0, 2, 1, 3, 4).reshape(B, hk, L, dk)
    v = (s["v_codes"][table][..., :dk, :] * s["v_scale"][table][..., None, None]).permute(0, 2, 1, 4, 3).reshape(B, hk, L, dk)
    n = cu[1:] - cu[:-1]
    row = torch.arange(R, device=q.device)
    source = (cu[:-1, None] + row[None]).clamp(max=q.shape[0] - 1)
    qp = q[source].reshape(B, R, hk, group, dk).permute(0, 2, 3, 1, 4).reshape(B, hk, group * R, dk)
    scores = torch.matmul(qp, k.transpose(2, 3)).mul_(s["scale"]).view(B, hk, group, R, L)
    key = torch.arange(L, device=q.device)
    last = (lens - n)[:, None] + row[None] if c["causal"] else (lens - 1)[:, None].expand(B, R)
    hidden = key[None, None] > torch.minimum(last, (lens - 1)[:, None])[..., None]          # [B, R, L]
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(top).exp_()
    out = torch.matmul(p.view(B, hk, group * R, L), v).view(B, hk, group, R, dk) / p.sum(-1, keepdim=True)
    out = out.permute(0, 3, 1, 2, 4).reshape(B, R, c["heads"], dk)
    keep = row[None] < n[:, None]
    return out[keep].to(s["q"].dtype)


def _plain_codes(x, slots, codes, scale, block, width):
    """``x`` [n, kv_heads, dk] into codes [blocks, kv_heads, block, width] in 64 bits: a block's scale is its
    largest magnitude / 127 and only grows, until the block is begun again at its first place."""
    dk = x.shape[-1]
    at, place = slots // block, slots % block
    first = torch.full((codes.shape[0],), block, dtype=torch.long, device=x.device).scatter_reduce(0, at, place, "amin")
    kept = torch.arange(block, device=x.device)[None] < first[:, None]                       # [blocks, block]
    top = torch.zeros_like(scale).scatter_reduce(0, at[:, None].expand(-1, scale.shape[1]), x.float().abs().amax(-1), "amax")
    before = torch.where(first[:, None] == 0, torch.zeros_like(scale), scale)
    touched = (first < block)[:, None]
    after = torch.where(touched, torch.maximum(before, (top.double() / 127).float()), scale)
    fresh = touched & (after > before)
    s64 = after.double()
    safe = torch.where(s64 == 0, torch.ones_like(s64), s64)
    old = (codes.double() * before.double()[..., None, None] / safe[..., None, None]).round().to(torch.int8)
    codes = torch.where((fresh[..., None] & kept[:, None])[..., None], old, codes)
    mine = safe[at][..., None]
    new = torch.where(after[at][..., None] == 0, torch.zeros_like(mine), x.double() / mine).round().clamp(-127, 127)
    padded = torch.zeros((x.shape[0], x.shape[1], width), dtype=torch.int8, device=x.device)
    padded[..., :dk] = new.to(torch.int8)
    codes[at, :, place] = padded
    return codes, after


def _plain_append(s):
    block, width = s["k_codes"].shape[2], s["k_codes"].shape[3]
    slots = s["slots"].long()
    k, ks = _plain_codes(s["k"], slots, s["k_codes"], s["k_scale"], block, width)
    v, vs = _plain_codes(s["v"], slots, s["v_codes"].transpose(2, 3), s["v_scale"], block, width)
    return k, v.transpose(2, 3), ks, vs


def _plain_plan(s):
    c = s["case"]
    block, W, B = c["block"], c["table"], c["batch"]
    lens, new, free = s["lens"].long(), s["new_rows"].long(), s["free_blocks"]
    gone = new < 0
    n = new.clamp(min=0)
    have = (lens + block - 1) // block
    # blocks of finished requests go on top of the stack, in order
    freed = torch.where(gone, have, torch.zeros_like(have))
    base = s["free_count"].long() + freed.cumsum(0) - freed
    column = torch.arange(W, device=lens.device)
    place = torch.where(gone[:, None] & (column[None] < have[:, None]), base[:, None] + column[None], free.shape[0])
    stack = torch.cat([free, free[:1]]).scatter(0, place.reshape(-1), s["tables"].reshape(-1))[:-1]
    level = s["free_count"].long() + freed.sum()
    # new blocks come from the top
    need = torch.where(gone, torch.zeros_like(have), (lens + n + block - 1) // block - have)
    offset = need.cumsum(0) - need
    j = torch.arange((c["rows"] + block - 1) // block + 1, device=lens.device)
    taken = stack[(level - 1 - (offset[:, None] + j[None])).clamp(min=0)]
    target = torch.where(j[None] < need[:, None], have[:, None] + j[None], W)
    tables = torch.cat([s["tables"], s["tables"][:, :1]], 1).scatter(1, target, taken)[:, :-1].contiguous()
    cu = torch.cat([torch.zeros_like(n[:1]), n.cumsum(0)])
    t = torch.arange(s["rows"], device=lens.device)
    b = (torch.searchsorted(cu, t, right=True) - 1).clamp(max=B - 1)
    pos = lens[b] + t - cu[b]
    used = t < cu[-1]
    pos = torch.where(used, pos, torch.zeros_like(pos))
    slots = torch.where(used, tables[b, pos // block].long() * block + pos % block, torch.full_like(pos, -1))
    lens_out = torch.where(gone, torch.zeros_like(lens), lens + n)
    i = torch.int32
    return cu.to(i), slots.to(i), pos.to(i), lens_out.to(i), (level - need.sum()).to(i).reshape(1), tables, stack


def _plain_logits(s):
    x = s["logits"].float()
    R, V = x.shape
    ids = s["history"].long()
    live = torch.arange(ids.shape[1], device=x.device)[None] < s["history_len"][:, None]
    count = torch.zeros((R, V + 1), device=x.device).scatter_add_(1, torch.where(live, ids, V), torch.ones_like(ids, dtype=torch.float32))[:, :V]
    seen = count > 0
    rep = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][:, None] * count - s["presence"][:, None] * seen
    if s["bias_ids"] is not None:
        b = s["bias_ids"].long()
        bias = torch.zeros((R, V + 1), device=x.device).scatter_add_(1, torch.where(b >= 0, b, V), s["bias_values"])
        x = x + bias[:, :V]
    if s["allowed"] is not None:
        cls = torch.arange(V, device=x.device)
        bits = (s["allowed"][:, cls // 32] >> (cls % 32)[None]) & 1
        x = torch.where(bits == 1, x, torch.full_like(x, -math.inf))
    return x.to(s["logits"].dtype)


def _values(k_codes, v_codes, k_scale, v_scale):
    """What the codes stand for."""
    return k_codes * k_scale[..., None, None], v_codes * v_scale[..., None, None], k_scale, v_scale


# ------------------------------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if own:
        from athena_amd import ops
        s = state
        if op == "attention":
            return ops.kv8_attention(s["q"], s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"], s["tables"], s["lens"],
                                     cu_rows=s["cu_rows"], max_rows=s["max_rows"], causal=s["case"]["causal"], scale=s["scale"])
        if op == "append":
            # (a pass repeated on the same state finds the scales grown by the first, and writes the same codes)
            ops.kv8_append(s["k"], s["v"], s["slots"], s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"])
            return _values(s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"])
        if op == "plan":
            p = ops.kv_plan(s["lens"], s["new_rows"], s["tables"], s["free_blocks"], s["free_count"], s["case"]["block"],
                            s["rows"], in_place=False)
            return p.cu_rows, p.slots, p.positions, p.lens, p.free_count, s["tables"], s["free_blocks"]
        return ops.logits_process(s["logits"], history=s["history"], history_len=s["history_len"], repetition=s["repetition"],
                                  presence=s["presence"], frequency=s["frequency"], bias_ids=s["bias_ids"],
                                  bias_values=s["bias_values"], allowed=s["allowed"])
    if op == "attention":
        return _plain_attention(state)
    if op == "append":
        return _values(*_plain_append(state))
    return _plain_plan(state) if op == "plan" else _plain_logits(state)


# ------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    size = {"bf16": 2, "fp32": 4}
    if case["op"] == "attention":
        lens = _lens(case)
        rows = _rows(case, lens)
        block, hk, dk, h = case["block"], case["kv_heads"], case["head_size"], case["heads"]
        cached = lens[:1] if case["shared"] else lens
        blocks = sum(-(-n // block) for n in cached)
        pairs = sum(_visible(n, r, case["causal"]) for n, r in zip(lens, rows))
        return {"bytes": 2 * sum(cached) * hk * dk + 8 * blocks * hk + 4 * blocks + 2 * sum(rows) * h * dk * size[case["dtype"]],
                "flops": 4.0 * pairs * h * dk}
    if case["op"] == "append":
        values = 2 * case["tokens"] * case["kv_heads"] * case["head_size"]
        return {"bytes": values * (size[case["dtype"]] + 1) + 4 * case["tokens"], "flops": 2.0 * values}
    if case["op"] == "plan":
        lens, new = _plan_sizes(case)
        block = case["block"]
        moved = sum(-(-n // block) if r < 0 else -(-(n + r) // block) - -(-n // block) for n, r in zip(lens, new))
        rows = sum(max(r, 0) for r in new) + 5
        return {"bytes": 16.0 * case["batch"] + 8.0 * moved + 8.0 * rows, "flops": 1.0 * rows}
    R, V = case["rows"], case["vocab"]
    used = sum(_spread(max(1, case["history"] // 4), case["history"], R))
    return {"bytes": 2.0 * R * V * size[case["dtype"]] + 4.0 * used + 8.0 * R * case["biases"] + (R * V / 8.0 if case["masked"] else 0),
            "flops": 4.0 * R * V}


# ------------------------------------------------------------------------------------------ 64 bits
def _code_width(s):
    return s["k_codes"].shape[3]


def _exact_attention(s):
    c = s["case"]
    lens = s["lens"].tolist()
    cu = s["cu_rows"].tolist() if s["cu_rows"] is not None else list(range(c["batch"] + 1))
    block, hk, dk, group = c["block"], c["kv_heads"], c["head_size"], c["heads"] // c["kv_heads"]
    out = torch.zeros((cu[-1], c["heads"], dk), dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        blocks = s["tables"][b, :-(-n // block)].long()
        r = cu[b + 1] - cu[b]
        for h in range(hk):
            k = (s["k_codes"][blocks, h].double() * s["k_scale"][blocks, h].double()[:, None, None]).reshape(-1, _code_width(s))[:n, :dk]
            v = (s["v_codes"][blocks, h].double() * s["v_scale"][blocks, h].double()[:, None, None]).transpose(1, 2).reshape(-1, _code_width(s))[:n, :dk]
            q = s["q"][cu[b]:cu[b + 1], h * group:(h + 1) * group].double().reshape(r * group, dk)
            w = q @ k.t() * s["scale"]
            if c["causal"] and r > 1:
                own_place = n - r + torch.arange(r, device="cuda").repeat_interleave(group)
                w[torch.arange(n, device="cuda")[None] > own_place[:, None]] = -math.inf
            out[cu[b]:cu[b + 1], h * group:(h + 1) * group] = (torch.softmax(w, -1) @ v).reshape(r, group, dk)
    return out


def _exact_append(s):
    """Block by block: the values that a block stands for when its rows are in."""
    block = s["k_codes"].shape[2]
    dk = s["k"].shape[2]
    slots = s["slots"].tolist()
    runs = []                                               # (block, first place, first row, rows)
    for i, slot in enumerate(slots):
        if runs and runs[-1][0] == slot // block:
            runs[-1][3] += 1
        else:
            runs.append([slot // block, slot % block, i, 1])
    got = []
    for x, codes, scale in ((s["k"], s["k_codes"], s["k_scale"]), (s["v"], s["v_codes"].transpose(2, 3), s["v_scale"])):
        codes, scale = codes.double().clone(), scale.clone()
        for at, place, i, n in runs:
            rows = x[i:i + n].double().transpose(0, 1)      # [kv_heads, n, dk]
            old = scale[at] if place else torch.zeros_like(scale[at])
            new = torch.maximum(old, (rows.abs().amax((1, 2)) / 127).float())
            if place:
                grown = torch.round(codes[at, :, :place] * old.double()[:, None, None] / new.double()[:, None, None])
                codes[at, :, :place] = torch.where((new > old)[:, None, None], grown, codes[at, :, :place])
            codes[at, :, place:place + n] = 0
            codes[at, :, place:place + n, :dk] = torch.round(rows / new.double()[:, None, None]).clamp(-127, 127)
            scale[at] = new
        got.append((codes * scale.double()[..., None, None], scale.double()))
    (k, ks), (v, vs) = got
    return k, v.transpose(2, 3), ks, vs


def _exact_logits(s):
    x = s["logits"].double()
    R, V = x.shape
    for r in range(R):
        ids, n = torch.unique(s["history"][r, :int(s["history_len"][r])].long(), return_counts=True)
        old = x[r, ids]
        rep = s["repetition"][r].double()
        x[r, ids] = torch.where(old > 0, old / rep, old * rep) - s["frequency"][r].double() * n - s["presence"][r].double()
        if s["bias_ids"] is not None:
            b = s["bias_ids"][r].long()
            x[r].index_add_(0, b[b >= 0], s["bias_values"][r].double()[b >= 0])
    if s["allowed"] is not None:
        shift = torch.arange(32, device="cuda", dtype=torch.int32)
        bits = ((s["allowed"][..., None] >> shift) & 1).reshape(R, -1)[:, :V]
        x[bits == 0] = -math.inf
    return x


def exact(case, seed):
    if case["op"] == "plan":
        return None                                         # whole numbers: they are equal or wrong
    s = prepare(case, seed)
    return {"attention": _exact_attention, "append": _exact_append, "logits": _exact_logits}[case["op"]](s)
