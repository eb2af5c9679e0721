"""Decoding with the 8-bit key / value cache: the cached step against the whole-history step, beam search with it,
and with penalties and a grammar.

A cached element is off by at most half a step, 1/254 of its block's largest; with the largest about 2.5 deviations
out that is 2.5 / 254 / sqrt(3) = 0.6 % rms of the keys and values.  A logit is a sum over many of them: 3 % of the
logits' scale is five of those deviations, and a wrong position, parent or block moves logits by their whole scale."""
import numpy as np
import pytest
import torch

from oracle import decode as od
from oracle import model as om
from tests.modelutil import model_config
from tests.test_decode_gpu import CASE, _one, _trained
from tests.test_model_gpu import build, oracle_params
from tests.util import assert_close

pytestmark = pytest.mark.gpu
TOL = 3e-2


@pytest.mark.parametrize("precision", ["fp32", "bf16"])
@pytest.mark.parametrize("graph", [True, False])
@pytest.mark.parametrize("mc", [model_config(32, 16, 4, 2, 2, 64), model_config(64, 16, 4, 1, 3, 96), model_config(256, 16, 4, 1, 2, 512)])
def test_cached_steps_match_the_whole_history(precision, mc, graph):
    from athena_amd import CachedPropagate
    case = dict(CASE, mc=mc)
    model, samples, _ = build(case, precision)
    ds = model.prepare_samples(_one(samples, 1))
    enc = model.model.decode(ds, None, None, return_encoder=True)
    step = CachedPropagate(model, 3, graph=graph)
    step.begin(*enc, max_labels=40)
    g = np.random.default_rng(3)
    seqs = np.array([[9]])
    grow = lambda s, parents: np.concatenate([s[parents], g.integers(1, 9, size=(len(parents), 1))], axis=1)
    # a beam that opens, keeps its order, swaps, drops a row and takes one twice; past a block's end
    moves = [None, [0, 0, 0], [0, 1, 2], [2, 0, 1], [0, 1], [1, 1, 0], [0, 2, 2]] + [[1, 0, 2], [0, 1, 2]] * 7
    for parents in moves:
        if parents is not None:
            seqs = grow(seqs, parents)
        want, _, _ = model.time_propagate([], torch.tensor(seqs), seqs.shape[1] - 1, enc)
        got, hist, after = step([], seqs, seqs.shape[1] - 1, enc)
        assert after == seqs.shape[1] and len(hist) == 1 and got.dtype == torch.float32
        assert_close(got, want.cpu(), TOL if precision == "fp32" else 2 * TOL, "step %d" % seqs.shape[1])
    assert int(step.free_count) == step.free_blocks.numel() - 3 * -(-seqs.shape[1] // 16)
    # hypotheses that extend nothing are computed afresh, and the next step goes on from them
    seqs = g.integers(1, 9, size=(2, 7))
    for _ in range(2):
        got, _, _ = step([], seqs, 0, enc)
        want, _, _ = model.time_propagate([], torch.tensor(seqs), seqs.shape[1] - 1, enc)
        assert_close(got, want.cpu(), TOL if precision == "fp32" else 2 * TOL, "afresh")
        seqs = grow(seqs, [1, 0])
    assert any(step.recorded.values()) == graph
    # another utterance, the recorded steps of the first still in use
    enc = model.model.decode(model.prepare_samples(_one(samples, 2)), None, None, return_encoder=True)
    step.begin(*enc, max_labels=40)
    seqs = np.array([[9]])
    for parents in ([0, 0, 0], [2, 2, 1], [0, 1, 2]):
        want, _, _ = model.time_propagate([], torch.tensor(seqs), seqs.shape[1] - 1, enc)
        got, _, _ = step([], seqs, seqs.shape[1] - 1, enc)
        assert_close(got, want.cpu(), TOL if precision == "fp32" else 2 * TOL, "next utterance, step %d" % seqs.shape[1])
        seqs = grow(seqs, parents)
    with pytest.raises(RuntimeError):
        step([], g.integers(1, 9, size=(4, 3)), 0, enc)
    with pytest.raises(RuntimeError):
        step([], g.integers(1, 9, size=(1, step.room + 1)), 0, enc)


def test_longer_utterances_keep_most_of_what_is_recorded():
    """Tolerances as above; room for 24 labels and 20 frames is 32 of each, and grows to twice that at least."""
    from athena_amd import CachedPropagate
    model, samples, _ = build(dict(CASE, mc=model_config(64, 16, 4, 1, 3, 96)), "fp32")
    enc, mask = model.model.decode(model.prepare_samples(_one(samples, 1)), None, None, return_encoder=True)
    enc = torch.cat([enc] * 8, dim=1)
    step = CachedPropagate(model, 2)
    seen = []
    for T, labels, room in ((20, 24, 32), (30, 30, 32), (33, 24, 32), (40, 40, 64), (50, 64, 64), (63, 65, 128)):
        frames = (enc[:, :T].contiguous(), None)
        step.begin(*frames, max_labels=labels)
        assert step.room == room and step.memory_frames == (32 if T < 33 else 64)
        if not any(r is step.recorded for r in seen):
            seen.append(step.recorded)
        seqs = np.array([[9], [9]])
        for i in range(4):
            want, _, _ = model.time_propagate([], torch.tensor(seqs), i, frames)
            got, _, _ = step([], seqs, i, frames)
            assert_close(got, want.cpu(), TOL, "%d frames, step %d" % (T, i))
            seqs = np.concatenate([seqs, [[1 + i], [2 + i]]], axis=1)
    assert len(seen) <= 4


def _score(p, ocfg, mem, mask, hyp):
    """Log-probability per label of a hypothesis (with its <eos>) in 64 bits."""
    sos = ocfg["num_class"] - 1
    total = 0.0
    for i, label in enumerate(hyp):
        total += float(torch.log_softmax(od.decoder_step(p, ocfg, [[sos] + hyp[:i]], mem, mask)[0], -1)[label])
    return total / (len(hyp) + 1)


@pytest.mark.parametrize("beam_size,ctc_weight", [(1, 0.0), (4, 0.0), (4, 0.3)])
def test_beam_search_with_the_cache(beam_size, ctc_weight):
    from athena_amd import DecoderSolver
    model, samples, ocfg = _trained()
    p = oracle_params(model)
    config = {"decoder_type": "beam_search_decoder", "beam_size": beam_size, "ctc_weight": ctc_weight, "lm_weight": 0.0}
    plain, cached = DecoderSolver(model, config=config), DecoderSolver(model, config=dict(config, kv_cache=True))
    for i in range(CASE["B"]):
        s1 = _one(samples, i)
        ds = model.prepare_samples(s1)
        want = model.decode(ds, plain.hparams, plain.decoder)[0].tolist()
        got = model.decode(ds, cached.hparams, cached.decoder)[0].tolist()
        assert got[-1] == ocfg["num_class"] - 1
        if got != want and ctc_weight == 0.0:
            # another hypothesis only where the two are as good as each other (beam 1: greedy, no such bound)
            s64 = {k: (v.double() if v.is_floating_point() else v) for k, v in s1.items()}
            with torch.no_grad():
                mem, mask = od.encode(p, s64, ocfg)
                assert beam_size == 1 or _score(p, ocfg, mem, mask, got) > _score(p, ocfg, mem, mask, want) - 0.1
    data = [_one(samples, i) for i in range(CASE["B"])]
    assert abs(cached.inference(data) - plain.inference(data)) <= 0.25


@pytest.mark.parametrize("kv_cache", [False, True])
def test_beam_search_with_penalties_biases_and_a_grammar(kv_cache):
    from athena_amd import DecoderSolver, LogitRules
    model, samples, ocfg = _trained(steps=40)
    eos, V = ocfg["num_class"] - 1, ocfg["num_class"]
    ds = model.prepare_samples(_one(samples, 0))
    config = {"decoder_type": "beam_search_decoder", "beam_size": 3, "ctc_weight": 0.0, "lm_weight": 0.0, "kv_cache": kv_cache}

    def decode(rules=None, **more):
        solver = DecoderSolver(model, config=dict(config, **more))
        if rules is not None:
            solver.decoder.set_logit_rules(rules)
        return model.decode(ds, solver.hparams, solver.decoder)[0].tolist()

    # a frequency penalty beyond any difference of logits: no label comes twice
    out = decode(frequency_penalty=1e4)
    assert len(set(out)) == len(out)
    # a bias that decides everything, and its opposite
    assert decode(LogitRules(bias={eos: 1e4})) == [eos]
    assert 5 not in decode(LogitRules(bias={5: -1e4}))

    def alternate(seqs):
        """Odd labels after even ones and the other way round; <eos> after four labels."""
        allowed = np.zeros((len(seqs), V), dtype=bool)
        for row, s in zip(allowed, seqs):
            if len(s) > 4:
                row[eos] = True
            else:
                row[1 - s[-1] % 2:eos:2] = True
                row[0] = False
        return allowed

    out = decode(LogitRules(grammar=alternate))
    assert len(out) == 5 and out[-1] == eos and all((a + b) % 2 for a, b in zip([eos] + out, out[:4]))


@pytest.mark.parametrize("graph", [True, False])
def test_labels_that_there_are_not(graph):
    """time_propagate takes them for the nearest label; here they must not be looked up outside the table.  Tolerances as above."""
    from athena_amd import CachedPropagate
    model, samples, ocfg = build(dict(CASE, mc=model_config(64, 16, 4, 1, 2, 96)), "fp32")
    enc = model.model.decode(model.prepare_samples(_one(samples, 1)), None, None, return_encoder=True)
    step = CachedPropagate(model, 2, graph=graph)
    step.begin(*enc, max_labels=20)
    V = ocfg["num_class"]
    seqs = np.array([[V - 1, -3], [V + 5, 2]])
    for new in ([V, -1], [2 ** 30, 1], [-2 ** 31, 2 ** 31 - 1], [3, 4]):
        want, _, _ = model.time_propagate([], torch.tensor(seqs), seqs.shape[1] - 1, enc)
        got, _, _ = step([], seqs, seqs.shape[1] - 1, enc)
        assert_close(got, want.cpu(), TOL, "step %d" % seqs.shape[1])
        seqs = np.concatenate([seqs, np.array(new)[:, None]], axis=1)


def test_memory_masks_with_holes_are_refused():
    """A cache has a length: what a mask leaves must be the first frames, one at least.  Tolerances as above."""
    from athena_amd import CachedPropagate
    model, samples, _ = build(dict(CASE, mc=model_config(64, 16, 4, 1, 2, 96)), "fp32")
    enc, _ = model.model.decode(model.prepare_samples(_one(samples, 1)), None, None, return_encoder=True)
    T = enc.shape[1]
    step = CachedPropagate(model, 2)
    for hidden in ([0], range(T), [1], [T - 2], range(1, T - 1)):
        mask = torch.zeros(1, 1, 1, T, device=enc.device)
        mask[..., list(hidden)] = 1
        with pytest.raises(RuntimeError, match="mask"):
            step.begin(enc, mask, max_labels=20)
    with pytest.raises(RuntimeError, match="mask"):
        step.begin(enc, torch.zeros(1, 1, 1, T - 1, device=enc.device), max_labels=20)
    for frames in (1, T - 1, T):
        mask = torch.zeros(1, 1, 1, T, device=enc.device)
        mask[..., frames:] = 1
        step.begin(enc, mask, max_labels=20)
        seqs = np.array([[9, 1], [9, 2]])
        want, _, _ = model.time_propagate([], torch.tensor(seqs), 1, (enc, mask))
        got, _, _ = step([], seqs, 1, (enc, mask))
        assert_close(got, want.cpu(), TOL, "%d frames" % frames)
