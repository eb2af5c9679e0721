"""What the decoding operators refuse, checked in front of any launch (no GPU is needed), and the loop
restatements the GPU tests compare with, checked against hand-made cases."""
import numpy as np
import pytest
import torch

from athena_amd import _lib, ops
from oracle import kv_cache as ok


def _cache(nb=4, hk=2, bs=16, w=32):
    return (torch.zeros(nb, hk, bs, w, dtype=torch.int8), torch.zeros(nb, hk, w, bs, dtype=torch.int8), torch.zeros(nb, hk),
            torch.zeros(nb, hk))


def _i(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


@pytest.mark.parametrize("change", ["codes_type", "codes_shape", "codes_strided", "scale_size", "scale_type", "heads", "head_size",
                                    "k_v_differ", "slots_type", "slots_short", "k_columns_strided"])
def test_append_refusals(change):
    kc, vc, ks, vs = _cache()
    k, v, slots = torch.zeros(3, 2, 24), torch.zeros(3, 2, 24), _i(3)
    if change == "codes_type": kc = kc.to(torch.uint8)
    if change == "codes_shape": vc = vc.transpose(2, 3).contiguous()
    if change == "codes_strided": kc = kc.transpose(0, 1)
    if change == "scale_size": ks = torch.zeros(4)
    if change == "scale_type": vs = vs.double()
    if change == "heads": k, v = torch.zeros(3, 3, 24), torch.zeros(3, 3, 24)
    if change == "head_size": k, v = torch.zeros(3, 2, 33), torch.zeros(3, 2, 33)
    if change == "k_v_differ": v = v.to(torch.bfloat16)
    if change == "slots_type": slots = slots.long()
    if change == "slots_short": slots = _i(2)
    if change == "k_columns_strided": k = torch.zeros(3, 2, 48)[..., ::2]
    with pytest.raises(RuntimeError, match="kv8_append"):
        ops.kv8_append(k, v, slots, kc, vc, ks, vs)


@pytest.mark.parametrize("change", ["heads", "head_size", "rows_without_cu", "cu_short", "tables_type", "tables_rows", "tables_strided",
                                    "lens_type", "out_shape", "out_type", "lse", "max_rows"])
def test_attention_refusals(change):
    kc, vc, ks, vs = _cache()
    q, tables, lens, kw = torch.zeros(3, 4, 32), _i(3, 2), _i(3), {}
    if change == "heads": q = torch.zeros(3, 3, 32)
    if change == "head_size": q = torch.zeros(3, 4, 33)
    if change == "rows_without_cu": q = torch.zeros(4, 4, 32)
    if change == "cu_short": kw = dict(cu_rows=_i(3))
    if change == "tables_type": tables = tables.long()
    if change == "tables_rows": tables = _i(2, 2)
    if change == "tables_strided": tables = _i(3, 4)[:, ::2]
    if change == "lens_type": lens = lens.long()
    if change == "out_shape": kw = dict(out=torch.zeros(3, 4, 16))
    if change == "out_type": kw = dict(out=torch.zeros(3, 4, 32, dtype=torch.bfloat16))
    if change == "lse": kw = dict(lse=torch.zeros(3, 4).double())
    if change == "max_rows": kw = dict(cu_rows=_i(4), max_rows=0)
    with pytest.raises(RuntimeError, match="kv8_attention"):
        ops.kv8_attention(q, kc, vc, ks, vs, tables, lens, **kw)


@pytest.mark.parametrize("change", ["lens_type", "new_short", "tables_rows", "free_type", "count_type"])
def test_plan_refusals(change):
    lens, new, tables, free, count = _i(3), _i(3), _i(3, 4), _i(8), _i(1)
    if change == "lens_type": lens = lens.long()
    if change == "new_short": new = _i(2)
    if change == "tables_rows": tables = _i(2, 4)
    if change == "free_type": free = free.float()
    if change == "count_type": count = count.long()
    with pytest.raises(RuntimeError, match="kv_plan"):
        ops.kv_plan(lens, new, tables, free, count, 16, 8)


@pytest.mark.parametrize("change", ["logits_dim", "logits_strided", "history_rows", "history_type", "len_type", "no_history", "repetition",
                                    "bias", "ids_alone", "allowed", "allowed_type", "out"])
def test_logits_refusals(change):
    x, kw = torch.zeros(2, 40), dict(history=_i(2, 5))
    if change == "logits_dim": x = torch.zeros(40)
    if change == "logits_strided": x = torch.zeros(2, 80)[:, ::2]
    if change == "history_rows": kw = dict(history=_i(3, 5))
    if change == "history_type": kw = dict(history=torch.zeros(2, 5))
    if change == "len_type": kw["history_len"] = torch.zeros(2, dtype=torch.int64)
    if change == "no_history": kw = dict(presence=torch.zeros(2))
    if change == "repetition": kw["repetition"] = torch.ones(3)
    if change == "bias": kw = dict(bias=torch.zeros(2, 39))
    if change == "ids_alone": kw = dict(bias_ids=_i(2, 1))
    if change == "allowed": kw = dict(allowed=_i(2, 1))
    if change == "allowed_type": kw = dict(allowed=torch.zeros(2, 2, dtype=torch.int64))
    if change == "out": kw["out"] = torch.zeros(2, 40, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="logits_process"):
        ops.logits_process(x, **kw)


def test_the_c_entries_refuse_before_any_launch():
    lib, p = _lib.load(), 4096                          # an address that is never followed
    attn = lambda bs=16, w=32, h=4, dk=32, dtype=0, q=p, nb=4, B=1, n=1, cu=0, mr=1, codes=p, W=1, ws=0: lib.athena_kv8_attention(
        _lib.Kv8AttentionDesc.pack(q, codes, p, p, p, p, p, cu, p, 0, ws, 0, 128, 32, 128, 32, W, dtype, nb, bs, w, W, B, mr, n, h, 2, dk, 1,
                                   1.0, 0.0), None)
    for kw in (dict(bs=24), dict(w=48), dict(h=3), dict(dk=33), dict(dk=0), dict(dtype=2), dict(q=0), dict(nb=0), dict(B=0),
               dict(B=70000), dict(cu=p, mr=0), dict(nb=1 << 28), dict(codes=4100), dict(n=2), dict(W=1 << 20), dict(W=1 << 27),
               dict(h=2, n=(1 << 31) - 100, cu=p)):
        assert attn(**kw) < 0, kw
        assert b"athena_kv8_attention" in lib.athena_last_error()
    assert lib.athena_kv8_attention(None, None) < 0 and lib.athena_kv8_attention_workspace_bytes(None) == 0
    append = lambda bs=16, w=32, dk=32, dtype=0, k=p, n=1, codes=p: lib.athena_kv8_append(
        _lib.Kv8AppendDesc.pack(k, p, p, codes, p, p, p, 64, 32, 64, 32, dtype, n, 4, 2, bs, dk, w, 0), None)
    for kw in (dict(bs=8), dict(w=256), dict(dk=64), dict(dtype=5), dict(k=0), dict(n=-1), dict(n=1 << 30), dict(codes=4097)):
        assert append(**kw) < 0, kw
        assert b"athena_kv8_append" in lib.athena_last_error()
    plan = lambda B=1, W=4, ld=4, free=4, bs=16, rows=1, lens=p: lib.athena_kv_plan(
        _lib.KvPlanDesc.pack(lens, p, p, p, p, p, p, p, p, p, p, p, ld, W, free, B, bs, rows, 0), None)
    for kw in (dict(B=0), dict(W=0), dict(ld=3), dict(free=0), dict(bs=20), dict(rows=-1), dict(lens=0), dict(W=1 << 27, ld=1 << 27),
               dict(W=(1 << 27) - 1, ld=1 << 27), dict(W=(1 << 24) - 1, ld=1 << 24, bs=128)):
        assert plan(**kw) < 0, kw
        assert b"athena_kv_plan" in lib.athena_last_error()
    logits = lambda R=1, V=40, ldl=40, dtype=0, x=p, nb=0, L=0: lib.athena_logits_process(
        _lib.LogitsDesc.pack(x, p, 0, 0, 0, 0, 0, 0, 0, 0, 0, ldl, 40, 0, 0, 0, 0, 0, dtype, R, V, L, nb, 0), None)
    for kw in (dict(R=-1), dict(V=0), dict(ldl=39), dict(dtype=3), dict(x=0), dict(nb=1), dict(R=70000), dict(L=(1 << 30) + 1), dict(nb=(1 << 30) + 1)):
        assert logits(**kw) < 0, kw
        assert b"athena_logits_process" in lib.athena_last_error()
    assert logits(R=0) == 0 and append(n=0) == 0


def test_attention_refuses_launches_of_too_many_threads():
    """2^32 threads and more.  Few rows: 65535 sequences x 128 kv heads x 4 tiles of 16
    rows are 2^25 workgroups of 256; many rows: 65528 x 8 heads x 64 tiles of 128 rows the same."""
    lib, p = _lib.load(), 4096                          # an address that is never followed
    attn = lambda B, h, hk, n, cu, mr: lib.athena_kv8_attention(
        _lib.Kv8AttentionDesc.pack(p, p, p, p, p, p, p, cu, p, 0, 0, 0, h * 32, 32, h * 32, 32, 1, 0, 4, 16, 32, 1, B, mr, n, h, hk, 32, 1,
                                   1.0, 0.0), None)
    for call in ((65535, 8192, 128, 65535, 0, 1), (65528, 8, 8, 1 << 20, p, 8192)):
        assert attn(*call) < 0, call
        assert b"too many workgroups" in lib.athena_last_error(), lib.athena_last_error()


def test_cache_width():
    assert [ops.kv8_width(n) for n in (1, 32, 33, 64, 65, 128)] == [32, 32, 64, 64, 128, 128]
    with pytest.raises(NotImplementedError):
        ops.kv8_width(129)


def test_oracle_plan_takes_and_gives_back():
    got = ok.plan([16, 5, 33], [1, -1, 0], [[3, -1, -1], [7, -1, -1], [1, 2, 4]], [9, -1, -1], 1, 16, 4)
    # request 1's block 7 goes on top of the stack and request 0 takes it at once
    assert got["cu_rows"] == [0, 1, 1, 1] and got["slots"] == [7 * 16, -1, -1, -1] and got["positions"] == [16, 0, 0, 0]
    assert got["lens"] == [17, 0, 33] and got["free_count"] == 1 and got["tables"][0] == [3, 7, -1]
    assert got["free_blocks"] == [9, 7, -1] and got["status"] == [0, 0, 0, 0]
    short = ok.plan([16], [17], [[3, -1, -1]], [9], 1, 16, 4)
    assert short["status"] == [1, 0, 13, 0] and short["lens"] == [16] and short["slots"] == [-1] * 4


def test_oracle_append_grows_a_scale():
    codes, scale = torch.zeros(1, 1, 16, 32, dtype=torch.int8), torch.full((1, 1), 99.0)
    ok.append(torch.tensor([[[127.0, -63.5, 1.0]]]), [0], codes, scale)      # begins the block: its old scale is gone
    assert float(scale) == 1.0 and codes[0, 0, 0, :4].tolist() == [127, -64, 1, 0]
    ok.append(torch.tensor([[[254.0, 3.0, -3.0]]]), [1], codes, scale)
    assert float(scale) == 2.0 and codes[0, 0, 0, :4].tolist() == [64, -32, 0, 0]
    assert codes[0, 0, 1, :4].tolist() == [127, 2, -2, 0]                     # 1.5 rounds to the even 2


def test_pack_classes():
    from athena_amd.tools import pack_classes
    import numpy as np
    allowed = np.zeros((2, 40), dtype=bool)
    allowed[0, [0, 31, 32, 39]] = True
    words = pack_classes(allowed)
    assert words.dtype == torch.int32 and tuple(words.shape) == (2, 2)
    assert words[0].tolist() == [1 - 2 ** 31, 1 | 1 << 7] and words[1].tolist() == [0, 0]
    with pytest.raises(ValueError):
        pack_classes(allowed[0])


def test_logit_rules_are_off_by_default():
    from athena_amd import LogitRules
    from athena_amd.solver import DecoderSolver
    from athena_amd.tools import BeamSearchDecoder
    from athena_amd.utils.hparam import register_and_parse_hparams
    assert not LogitRules() and LogitRules(repetition=1.2) and LogitRules(bias={3: 1.0}) and LogitRules(grammar=lambda s: None)
    with pytest.raises(ValueError):
        LogitRules(repetition=0)
    hp = register_and_parse_hparams(DecoderSolver.default_config, {"decoder_type": "beam_search_decoder"})
    assert hp.kv_cache is False
    assert BeamSearchDecoder.build_decoder(hp, 4, 3, 3, lambda *a: None).logit_rules is None
    hp.frequency_penalty = 0.5
    assert BeamSearchDecoder.build_decoder(hp, 4, 3, 3, lambda *a: None).logit_rules.frequency == 0.5


def test_a_hypothesis_that_nothing_may_follow_comes_last():
    """Classes 0 to 3 and <eos> = 4; nothing may follow label 2, which every step likes best.  The others' scores are those
    of the softmax, in fp32 sums of a few numbers: 1e-6."""
    from athena_amd.tools.beam_search import BeamSearchDecoder, CandidateHolder
    row = torch.tensor([0.0, 4.0, 5.0, 1.0, 3.0])

    def step(logits, seqs, states, enc):
        return row.expand(len(seqs), -1), list(logits), states

    def rules(logits, seqs):
        return torch.where(torch.as_tensor(seqs[:, -1:] == 2), -float("inf"), logits)

    dec = BeamSearchDecoder(5, 4, 4, beam_size=2)
    dec.decoder_one_step = step
    dec.set_logit_rules(rules)
    seqs = np.array([[4, 1], [4, 2]])
    scores, _, _ = dec.beam_search_score(CandidateHolder(seqs, [], [seqs], np.zeros(2, np.float32), np.arange(2)), None)
    want = row.double() - torch.logsumexp(row.double(), 0)
    assert np.abs(scores[0] - want.numpy()).max() < 1e-6 and np.isneginf(scores[1]).all()
    # alone <eos> costs 2.4; label 2 first (0.4) leads nowhere
    out = dec(np.array([[4]]), [seqs[:1]], 0, (torch.zeros(1, 6, 8), None))[0].tolist()
    assert out[-1] == 4 and 2 not in out


# ------------------------------------------------------------------------------------------ grammars narrower than the beam
def _search(grammar, frames, beam_size, row, ctc=None):
    """(result, hypotheses handed to the grammar, steps) of a search over classes 0 .. n - 2 and <eos> = n - 1, every step of which likes the
    classes as ``row`` does; ``grammar`` maps one hypothesis (a list that begins with <eos> for <sos>) to the classes it may go on with."""
    from athena_amd.tools.beam_search import BeamSearchDecoder
    eos, asked, steps = len(row) - 1, [], []

    def step(logits, seqs, states, enc):
        steps.append(len(seqs))
        return torch.tensor(row).expand(len(seqs), -1), list(logits), states

    def rules(logits, seqs):
        allowed = torch.zeros(len(seqs), len(row), dtype=torch.bool)
        for r, s in zip(allowed, seqs.tolist()):
            asked.append(s)
            r[list(grammar(s))] = True
        return torch.where(allowed, logits, -float("inf"))

    dec = BeamSearchDecoder(len(row), eos, eos, beam_size=beam_size)
    dec.decoder_one_step = step
    dec.set_logit_rules(rules)
    start = np.array([[eos]])
    states = [start]
    if ctc is not None:
        from athena_amd import CTCPrefixScorer
        scorer = CTCPrefixScorer(eos, ctc_beam=2 * beam_size, num_classes=len(row), ctc_weight=0.3)
        dec.set_ctc_scorer(scorer)
        states = scorer.initial_state(states, ctc)
    return dec(start, states, 0, (torch.zeros(1, frames, 8), None))[0].tolist(), asked, steps


@pytest.mark.parametrize("with_ctc", [False, True])
@pytest.mark.parametrize("beam_size", [1, 4, 10])
def test_search_under_a_grammar_of_one_path(beam_size, with_ctc):
    """One path of three labels and <eos>, labels that every step likes least; the search ends with it."""
    path = [5, 0, 1, 3, 5]
    follow = lambda s: {path[len(s)]} if s == path[:len(s)] and len(s) < 5 else set()
    ctc = torch.log_softmax(torch.randn(1, 12, 6, generator=torch.Generator().manual_seed(1)), -1) if with_ctc else None
    out, asked, steps = _search(follow, 12, beam_size, [-3.0, -4.0, 6.0, -5.0, 5.0, 4.0], ctc)
    assert out == path[1:] and steps == [1, 1, 1, 1]
    assert asked == [path[:n] for n in range(1, 5)]


@pytest.mark.parametrize("beam_size", [2, 3, 8])
def test_a_grammar_is_asked_about_nothing_that_it_forbade(beam_size):
    """Even labels follow odd ones and the other way round, at most two of three; <eos> from three labels on."""
    def follow(s):
        if len(s) == 1:
            return {0, 1}
        return {c for c in (0, 1, 2) if (c + s[-1]) % 2} | ({6} if len(s) > 3 else set())

    out, asked, steps = _search(follow, 9, beam_size, [1.0, 2.0, 0.5, 7.0, 6.0, 5.0, 0.0])
    assert out[-1] == 6 and len(out) > 3
    for s in asked + [[6] + out]:
        assert all(c in follow(s[:i]) for i, c in enumerate(s) if i), s
    assert max(steps) <= beam_size and steps[0] == 1


def test_a_search_that_nothing_allowed_can_finish():
    """No <eos> at all, and a path that is longer than the frames; in time it is found."""
    with pytest.raises(RuntimeError, match="rules"):
        _search(lambda s: {0, 1}, 6, 3, [1.0, 2.0, 0.0])
    path = [3, 0, 1, 2, 0, 3]
    follow = lambda s: {path[len(s)]} if len(s) < 6 else set()
    with pytest.raises(RuntimeError, match="rules"):
        _search(follow, 4, 3, [1.0, 2.0, 0.5, 0.0])
    # (the pool of finished hypotheses is as wide as there are frames: what ends on the last one comes without its <eos>, here as without rules)
    assert _search(follow, 5, 3, [1.0, 2.0, 0.5, 0.0])[0] == path[1:5]
    assert _search(follow, 6, 3, [1.0, 2.0, 0.5, 0.0])[0] == path[1:]
    with pytest.raises(RuntimeError, match="rules"):
        _search(lambda s: set(), 6, 3, [1.0, 2.0, 0.0])


def test_a_search_whose_rules_forbid_nothing_is_the_plain_one():
    from athena_amd.tools.beam_search import BeamSearchDecoder
    g = torch.Generator().manual_seed(4)
    table = torch.randn(40, 7, generator=g) * 2

    def step(logits, seqs, states, enc):
        return table[torch.as_tensor(seqs.sum(1) % 40)], list(logits), states

    for frames in (1, 2, 9):
        outs = []
        for rules in (None, lambda logits, seqs: logits):
            dec = BeamSearchDecoder(7, 6, 6, beam_size=3)
            dec.decoder_one_step = step
            dec.set_logit_rules(rules)
            outs.append(dec(np.array([[6]]), [np.array([[6]])], 0, (torch.zeros(1, frames, 8), None)).tolist())
        assert outs[0] == outs[1]


def test_append_refuses_launches_of_too_many_threads():
    """64 rows a workgroup of 256 threads: from 2^30 - 63 rows on these are 2^32 threads."""
    lib, p = _lib.load(), 4096                          # an address that is never followed
    for n in ((1 << 30) - 63, (1 << 30) - 1):
        assert -(-n // 64) * 256 >= 1 << 32
        assert lib.athena_kv8_append(_lib.Kv8AppendDesc.pack(p, p, p, p, p, p, p, 64, 32, 64, 32, 0, n, 4, 2, 16, 32, 32, 0), None) < 0
        assert b"N=" in lib.athena_last_error()


def test_attention_workspace_of_a_row_bound_below_the_truth():
    """``max_rows`` shapes the launch, so a call may name fewer rows than its sequences have: the workspace stays that of the rows there are."""
    lib = _lib.load()
    need = lambda B, mr, n, h=32, hk=8, dk=128, w=128, W=8192, bs=64, dtype=1: lib.athena_kv8_attention_workspace_bytes(
        _lib.Kv8AttentionDesc.pack(0, 0, 0, 0, 0, 0, 0, 4096, 0, 0, 0, 0, h * dk, dk, h * dk, dk, W, dtype, 4, bs, w, W, B, mr, n, h, hk, dk, 1,
                                   1.0, 0.0))
    for B, n in ((1, 100000), (1, 2000000), (16, 500000), (65535, 4000000)):
        for mr in (1, 2, 15, 17, 100, 600, 4096):
            for dtype in (0, 1):
                for h, hk, dk, w in ((32, 8, 128, 128), (4, 4, 64, 64), (64, 1, 128, 128), (1, 1, 24, 32)):
                    assert need(B, mr, n, h, hk, dk, w, dtype=dtype) <= 204 << 20, (B, mr, n, h, hk)
    # rows as they are named: splits that fill the chip about three times over, B x kv heads x tiles of 16 rows
    assert need(64, 1, 64) == ((1535 + 512) // 512) * 64 * 32 * 129 * 4
    assert need(8, 1, 8) == ((1535 + 64) // 64) * 8 * 32 * 129 * 4
    assert need(1, 1, 1) == ((1535 + 8) // 8) * 32 * 129 * 4
