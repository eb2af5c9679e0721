"""Decoding operators on the GPU against loop restatements in whole numbers and 64 bits (oracle/kv_cache.py)."""
import math

import pytest
import torch

from athena_amd import ops
from oracle import kv_cache as ok
from tests.util import dev

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _i32(x):
    return torch.as_tensor(x, dtype=torch.int32).to(dev())


# ------------------------------------------------------------------------------------------ plans
def _plan_case(seed, B, width, bs, most, finished, spare=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=g))
    lens = [r(0, width * bs - most) for _ in range(B)]
    new = [-1 if r(1, 100) <= finished else r(0, most) for _ in range(B)]
    have = [-(-n // bs) for n in lens]
    pool = sum(have) + sum(-(-(n + max(m, 0)) // bs) for n, m in zip(lens, new)) - sum(have) + 5
    order = torch.randperm(pool, generator=g).tolist()
    tables, at = [], 0
    for h in have:
        tables.append(order[at:at + h] + [-1] * (width - h))
        at += h
    free = order[at:] + [-1] * at
    return lens, new, tables, free, pool - at, sum(max(m, 0) for m in new) + spare


def _run_plan(lens, new, tables, free, count, bs, rows, in_place=True):
    t, f, l, c = _i32(tables), _i32(free), _i32(lens), _i32([count])
    p = ops.kv_plan(l, _i32(new), t, f, c, bs, rows, in_place=in_place)
    if in_place:
        assert p.lens.data_ptr() == l.data_ptr() and p.free_count.data_ptr() == c.data_ptr()
    return dict(cu_rows=p.cu_rows.tolist(), slots=p.slots.tolist(), positions=p.positions.tolist(), lens=p.lens.tolist(),
                free_count=int(p.free_count), tables=t.tolist(), free_blocks=f.tolist(), status=p.status.tolist())


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("B,width,bs,most,finished,spare", [
    (1, 1, 16, 1, 0, 0), (1, 4, 64, 100, 0, 3), (7, 9, 16, 1, 30, 2), (64, 17, 32, 40, 50, 0), (65, 5, 128, 300, 10, 11),
    (1000, 12, 16, 3, 20, 1), (1025, 6, 16, 20, 50, 0), (3000, 4, 16, 9, 100, 4), (2500, 40, 16, 33, 5, 100)])
def test_plan(B, width, bs, most, finished, spare, in_place):
    case = _plan_case(B, B, width, bs, most, finished, spare)
    assert _run_plan(*case[:5], bs, case[5], in_place) == ok.plan(*case[:5], bs, case[5])


@pytest.mark.parametrize("what", ["blocks", "table", "negative", "rows", "stack"])
def test_a_plan_that_does_not_fit_changes_nothing(what):
    lens, new, tables, free, count, rows = _plan_case(3, 20, 9, 16, 30, 20, 0)
    if what == "blocks": count = 1
    if what == "table": new[4] = 9 * 16 + 1
    if what == "negative": lens[3] = -5
    if what == "rows": rows -= 1
    if what == "stack": free, count, new = free[:8], 8, [-1] * 20
    got = _run_plan(lens, new, tables, free, count, 16, rows)
    assert got == ok.plan(lens, new, tables, free, count, 16, rows)
    assert any(got["status"]) and got["lens"] == lens and got["tables"] == tables and got["free_blocks"] == free


def test_plan_huge_lengths_do_not_overflow():
    got = _run_plan([2 ** 31 - 1, 5], [2 ** 31 - 1, 1], [[0, -1], [1, -1]], [2], 1, 16, 4)
    assert got["status"] == [0, 1, 0, 0] and got["slots"] == [-1] * 4


def test_plan_without_room_for_rows_and_a_strided_table():
    wide = torch.full((2, 8), -1, dtype=torch.int32, device=dev())
    lens, free, count = _i32([0, 16]), _i32([5, 6]), _i32([2])
    wide[1, 0] = 3
    p = ops.kv_plan(lens, _i32([0, 0]), wide[:, :4], free, count, 16, 0)
    assert p.slots.numel() == 0 and p.cu_rows.tolist() == [0, 0, 0] and p.status.tolist() == [0] * 4
    p = ops.kv_plan(lens, _i32([1, 1]), wide[:, :4], free, count, 16, 2)
    assert wide.tolist() == [[6] + [-1] * 7, [3, 5] + [-1] * 6] and p.slots.tolist() == [96, 80] and int(count) == 0


# ------------------------------------------------------------------------------------------ writing
def _random_cache(g, nb, hk, bs, w, dk):
    kc = torch.randint(-127, 128, (nb, hk, bs, w), generator=g, dtype=torch.int8)
    vc = torch.randint(-127, 128, (nb, hk, w, bs), generator=g, dtype=torch.int8)
    kc[..., dk:] = 0
    vc[:, :, dk:] = 0
    ks, vs = (torch.exp(0.3 * torch.randn(nb, hk, generator=g)) / 40 for _ in range(2))
    return kc, vc, ks, vs


def _append_both(k, v, slots, cache):
    got = [t.to(dev()) for t in cache]
    ops.kv8_append(k if k.is_cuda else k.to(dev()), v if v.is_cuda else v.to(dev()), _i32(slots), *got)
    want = [t.clone() for t in cache]
    ok.append(k.cpu(), slots, want[0], want[2])
    vt = want[1].transpose(2, 3).contiguous()
    ok.append(v.cpu(), slots, vt, want[3])
    want[1] = vt.transpose(2, 3)
    return [t.cpu() for t in got], want


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("bs,hk,dk", [(16, 1, 8), (16, 3, 32), (32, 2, 64), (64, 2, 80), (128, 1, 128), (64, 4, 33)])
@pytest.mark.parametrize("rows", [1, 3, 50])
def test_append_codes_are_exact(dtype, bs, hk, dk, rows):
    g = torch.Generator().manual_seed(rows * 1000 + bs + dk)
    nb = 12
    # four sequences in different blocks that begin at different places, one in the middle of the rows skipped
    slots, at = [], 0
    for i in range(4):
        blocks = torch.randperm(3, generator=g).add(3 * i).tolist()
        first = [0, bs - 1, 5, bs // 2][i]
        n = min(rows, 3 * bs - first)
        slots += [blocks[(first + j) // bs] * bs + (first + j) % bs for j in range(n)]
        if i == 1:
            slots += [-1]
    k, v = (torch.randn(len(slots), hk, dk, generator=g).mul(2.0 ** (3 * j)).to(dtype) for j in range(2))
    got, want = _append_both(k, v, slots, _random_cache(g, nb, hk, bs, ops.kv8_width(dk), dk))
    for name, x, y in zip(("k_codes", "v_codes", "k_scale", "v_scale"), got, want):
        assert torch.equal(x, y), (name, (x != y).nonzero()[:5].tolist())


def test_append_values_on_and_next_to_rounding_borders():
    # the block's largest is 127: its scale is 1, and halves lie exactly on the borders; a scale that is no power of
    # two puts fp32 values next to borders
    g = torch.Generator().manual_seed(5)
    halves = torch.arange(-127, 127).float() + 0.5
    for top in (127.0, 3.3):
        s = (torch.tensor(top).double() / 127).float()
        x = torch.zeros(8, 1, 128)
        x[:, 0, 0] = top
        pick = halves[torch.randint(0, 254, (8, 127), generator=g)].double() * s.double()
        x[:, 0, 1:] = pick.float()
        x[1::3, 0, 1:] = torch.nextafter(x[1::3, 0, 1:], torch.tensor(math.inf))
        x[2::3, 0, 1:] = torch.nextafter(x[2::3, 0, 1:], torch.tensor(-math.inf))
        x.clamp_(-top, top)
        got, want = _append_both(x, -x, list(range(8)), _random_cache(g, 2, 1, 16, 128, 128))
        assert all(torch.equal(a, b) for a, b in zip(got, want)), top


def test_append_tiny_zero_and_not_finite_values():
    g = torch.Generator().manual_seed(6)
    for value in (0.0, 1e-45, 1e-42, 1e-38, 3e38):
        x = torch.full((3, 1, 32), value)
        x[1, 0, 3] = -value / 2
        for first in (0, 2):
            got, want = _append_both(x, x, [first, first + 1, first + 2], _random_cache(g, 2, 1, 16, 32, 32))
            assert all(torch.equal(a, b) for a, b in zip(got, want)), (value, first)
    for value in (math.inf, -math.inf, math.nan):
        x = torch.randn(3, 1, 32, generator=g)
        x[1, 0, 7] = value
        cache = _random_cache(g, 2, 1, 16, 32, 32)
        got, want = _append_both(x, x, [4, 5, 6], cache)
        assert not bool(torch.isfinite(got[2][0, 0])) and not bool(torch.isfinite(got[3][0, 0]))
        values = got[0].float() * got[2][..., None, None]
        assert bool(torch.isnan(values[0, 0, 4:7]).all()), "rows of that block stand for NaN"
        assert torch.equal(got[2][1], cache[2][1]) and torch.equal(got[0][1], cache[0][1]), "another block"
        # once not finite, until the block is begun again
        dev_cache = [t.to(dev()) for t in got]
        good = torch.randn(1, 1, 32, generator=g)
        ops.kv8_append(good.to(dev()), good.to(dev()), _i32([7]), *dev_cache)
        assert not bool(torch.isfinite(dev_cache[2][0, 0]))
        ops.kv8_append(good.to(dev()), good.to(dev()), _i32([0]), *dev_cache)
        assert float(dev_cache[2][0, 0]) == float((good.abs().max().double() / 127).float())


def test_append_strided_rows_many_rows_and_slots_outside():
    g = torch.Generator().manual_seed(7)
    bs, nb, hk, dk = 16, 200, 4, 64
    order = torch.randperm(nb, generator=g).tolist()
    slots = [order[i // bs] * bs + i % bs for i in range(2000)]
    for i in range(0, 2000, 97):
        slots[i] = [-1, nb * bs, 2 ** 31 - 1, -2 ** 31][i % 4]
    qkv = torch.randn(2000, 3, hk, dk, generator=g).to(BF16)
    whole = qkv.to(dev())
    cache = _random_cache(g, nb, hk, bs, 64, dk)
    # keys and values as column blocks of a fused projection
    got, want = _append_both(whole[:, 1], whole[:, 2], slots, cache)
    for x, y in zip(got, want):
        assert torch.equal(x, y)


def test_append_of_no_rows():
    cache = [t.to(dev()) for t in _random_cache(torch.Generator().manual_seed(1), 2, 1, 16, 32, 32)]
    before = [t.clone() for t in cache]
    ops.kv8_append(torch.zeros(0, 1, 32, device=dev()), torch.zeros(0, 1, 32, device=dev()), _i32([]), *cache)
    assert all(torch.equal(a, b) for a, b in zip(cache, before))


# ------------------------------------------------------------------------------------------ attention
def _attention_case(seed, lens, rows, h, hk, dk, bs, dtype, extra_width=1):
    g = torch.Generator().manual_seed(seed)
    need = [-(-max(n, 0) // bs) for n in lens]
    nb = sum(need) + 2
    order = torch.randperm(nb, generator=g).to(torch.int32)
    tables = torch.full((len(lens), max(need + [1]) + extra_width - 1), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = order[at:at + n]
        at += n
    cache = _random_cache(g, nb, hk, bs, ops.kv8_width(dk), dk)
    cu = [0]
    for r in rows:
        cu.append(cu[-1] + r)
    q = torch.randn(cu[-1], h, dk, generator=g).mul(0.5).to(dtype)
    return q, cache, tables, cu


def _bound(dtype, q, cache, spread, want, scale):
    """Half a step of the result's type, and what roundings inside leave: a score sums dk products in fp32 (each
    rounding 2^-24 of the sum of magnitudes; independent, so within 6 sqrt(dk + 8) of them), moves its probability by
    as much, and a probability times a value's scale is held in 11 bits (bf16 queries) or 22 (fp32): 2^-12 / 2^-22 of each term; sums over keys in
    fp32 add 2^-24 sqrt-wise, covered by the same 2^-21."""
    dk = q.shape[2]
    scales = torch.where(torch.isfinite(cache[2]), cache[2], 0)       # (blocks with others are not visible, or give NaN)
    kmax = float((cache[0].float().abs().amax((1, 2, 3)) * scales.amax(1)).max())
    score = float(q.double().abs().sum(-1).max()) * kmax * abs(scale)
    inner = 2 * 6 * math.sqrt(dk + 8) * 2.0 ** -24 * score + (2.0 ** -11 if dtype == BF16 else 2.0 ** -20)
    return torch.finfo(dtype).eps / 2 * want.abs() + inner * spread


def _check_attention(q, cache, tables, lens, cu, causal, dtype, scale=None, expand=False, max_rows=None, one_row=False, seed=0):
    n, h, dk = q.shape
    scale = scale if scale is not None else 1 / math.sqrt(dk)
    t = tables.to(dev())
    out = torch.full((n, h, dk), 7.0, dtype=dtype, device=dev())
    lse = torch.full((n, h), 7.0, device=dev())
    most = max([b - a for a, b in zip(cu, cu[1:])] + [1]) if max_rows is None else max_rows
    ops.kv8_attention(q.to(dev()), *[x.to(dev()) for x in cache], t, _i32(lens), cu_rows=None if one_row else _i32(cu), max_rows=most,
                      causal=causal, scale=scale, out=out, lse=lse)
    want, want_lse, spread = ok.attention(q, *cache, tables, lens, None if one_row else cu, causal, scale)
    got, got_lse = out.double().cpu(), lse.double().cpu()
    mine = ~torch.isnan(want)
    assert bool((got[~mine] == 7.0).all()), "rows of no sequence are left as they were"
    err = ((got - want).abs() - _bound(dtype, q, cache, spread, want, scale))[mine]
    assert bool((err <= 0).all()), float(err.max())
    seen = torch.isfinite(want_lse)
    assert bool((got_lse[~torch.isnan(want_lse) & ~seen] == -math.inf).all())
    assert bool(((got_lse - want_lse).abs()[seen] <= 2e-5 * (1 + want_lse.abs()[seen])).all())
    return out


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("h,hk,dk,bs", [(4, 4, 8, 16), (4, 4, 64, 16), (8, 2, 128, 64), (6, 2, 80, 32), (7, 1, 32, 128), (32, 2, 128, 16),
                                        (40, 2, 64, 64)])
def test_attention_of_single_rows(dtype, h, hk, dk, bs):
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 200, 257]
    q, cache, tables, cu = _attention_case(h + dk, lens, [1] * len(lens), h, hk, dk, bs, dtype)
    for causal in (True, False):
        _check_attention(q, cache, tables, lens, cu, causal, dtype, one_row=True)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("h,hk,dk,bs", [(4, 4, 64, 16), (6, 2, 128, 64), (5, 1, 24, 32)])
def test_attention_of_many_rows(dtype, causal, h, hk, dk, bs):
    lens = [70, 1, 33, 130, 16]
    rows = [70, 1, 20, 5, 16]
    q, cache, tables, cu = _attention_case(dk, lens, rows, h, hk, dk, bs, dtype)
    _check_attention(q, cache, tables, lens, cu, causal, dtype)


def test_attention_of_more_rows_than_tokens_and_of_none():
    # a length of zero, sequences without rows, rows in front of a sequence's first token, rows behind the last
    lens, rows = [0, 5, 40, 0, 9], [3, 12, 0, 0, 2]
    q, cache, tables, cu = _attention_case(3, lens, rows, 4, 2, 64, 16, BF16)
    more = torch.cat([q, torch.randn(6, 4, 64).to(BF16)])
    for causal in (True, False):
        out = _check_attention(more, cache, tables, lens, cu, causal, BF16)
        assert bool((out[:3] == 0).all()), "nothing to see: zeros"
        if causal:
            assert bool((out[3:10] == 0).all()), "rows in front of the sequence see nothing"


def test_attention_does_not_depend_on_the_row_bound():
    lens, rows = [90, 300, 18], [40, 7, 18]
    q, cache, tables, cu = _attention_case(4, lens, rows, 4, 2, 64, 32, F32)
    outs = [_check_attention(q, cache, tables, lens, cu, True, F32, max_rows=m) for m in (1, 40, 1000)]
    for o in outs[1:]:
        assert float((o - outs[0]).abs().max()) <= 2.0 ** -18 * float(outs[0].abs().max())


def test_attention_of_bad_tables_lengths_and_offsets_stays_inside():
    lens = [100, 100, 5000, -3]
    q, cache, tables, cu = _attention_case(5, [100] * 4, [1] * 4, 4, 2, 64, 16, BF16)
    nb = cache[0].shape[0]
    tables[0, 2] = -1                                       # blocks that hold nothing
    tables[1, 0], tables[1, 6] = nb, 2 ** 31 - 1
    tables[2, 1] = -2 ** 31
    _check_attention(q, cache, tables, lens, cu, True, BF16, one_row=True)
    _check_attention(q, cache, tables, lens, [0, 1, 2, 3, 900], True, BF16)      # an offset beyond the rows
    _check_attention(q, cache, torch.full_like(tables, -1), lens, cu, True, BF16, one_row=True)


def test_attention_leaves_masked_blocks_alone():
    """Scales of blocks nothing of which is visible may be anything, codes behind the last token too."""
    lens = [20, 33]
    q, cache, tables, cu = _attention_case(6, [64, 64], [1, 1], 4, 2, 64, 16, F32)
    want = _check_attention(q, cache, tables, lens, cu, True, F32, one_row=True)
    for b, n in enumerate(lens):
        for j in range(-(-n // 16), 4):
            for s, value in ((2, math.nan), (3, math.inf)):
                cache[s][tables[b, j].long()] = value
    got = _check_attention(q, cache, tables, lens, cu, True, F32, one_row=True)
    assert torch.equal(got, want)


def test_attention_not_finite_inputs_stay_with_their_rows():
    lens = [40, 40, 40]
    q, cache, tables, cu = _attention_case(7, lens, [1] * 3, 2, 2, 64, 16, F32)
    q[1, 0, 3] = math.nan
    cache[3][int(tables[2, 1]), 1] = math.nan
    out = ops.kv8_attention(q.to(dev()), *[x.to(dev()) for x in cache], tables.to(dev()), _i32(lens)).cpu()
    nan = torch.isnan(out)
    assert nan.any(-1).tolist() == [[False, False], [True, False], [False, True]] == nan.all(-1).tolist()


def test_attention_value_scales_of_very_different_sizes():
    lens = [80, 80]
    q, cache, tables, cu = _attention_case(8, lens, [1, 1], 2, 2, 64, 16, F32)
    for i, s in enumerate((1e-30, 1e30, 1e-38, 1.0, 3e-3)):
        cache[3][tables[0, i].long()] = s
        cache[3][tables[1, 4 - i].long()] = s
    _check_attention(q, cache, tables, lens, cu, True, F32, one_row=True)
    for scale_of_all in (1e-36, 1e34, 0.0):
        cache[3][:] = scale_of_all
        _check_attention(q, cache, tables, lens, cu, True, F32, one_row=True)


def test_attention_queries_of_extreme_sizes():
    lens = [50, 50, 50, 50]
    q, cache, tables, cu = _attention_case(9, lens, [1] * 4, 2, 2, 64, 16, F32)
    q[0] *= 1e-30
    q[1] *= 1e-42
    q[2] = 0
    q[3, :, 1:] *= 1e-6
    _check_attention(q, cache, tables, lens, cu, True, F32, one_row=True)
    _check_attention(q.to(BF16), cache, tables, lens, cu, True, BF16, one_row=True)
    # scores far apart: one key takes everything
    big = torch.randn(4, 2, 64, generator=torch.Generator().manual_seed(1)) * 1e6
    out = ops.kv8_attention(big.to(dev()), *[x.to(dev()) for x in cache], tables.to(dev()), _i32(lens)).cpu()
    want, _, _ = ok.attention(big, *cache, tables, lens, None, True, 0.125)
    assert float((out.double() - want).abs().max()) <= 2.0 ** -20 * float(want.abs().max())


def test_attention_of_shared_blocks_and_strided_operands():
    lens = [37] * 5
    q, cache, tables, cu = _attention_case(10, [37], [1], 4, 2, 64, 16, BF16)
    q = torch.randn(5, 3, 4, 64, generator=torch.Generator().manual_seed(2)).to(BF16)
    wide = torch.zeros(5, 8, 64, dtype=BF16, device=dev())
    args = [x.to(dev()) for x in cache]
    got = ops.kv8_attention(q.to(dev())[:, 1], *args, tables.to(dev()).expand(5, -1), _i32(lens), causal=False, out=wide[:, 2:6])
    want, _, spread = ok.attention(q[:, 1], *cache, tables.expand(5, -1), lens, None, False, 0.125)
    err = (got.double().cpu() - want).abs() - _bound(BF16, q[:, 1], cache, spread, want, 0.125)
    assert bool((err <= 0).all()), float(err.max())
    assert bool((wide[:, :2] == 0).all() and (wide[:, 6:] == 0).all())


@pytest.mark.parametrize("h,hk,dk,bs,n", [(8, 1, 128, 64, 20011), (4, 4, 64, 16, 9999), (16, 2, 64, 128, 40000)])
def test_attention_over_long_contexts(h, hk, dk, bs, n):
    """The key axis split over workgroups, against the same sum in 64 bits on the GPU's codes."""
    lens = [n, 1, n // 3]
    q, cache, tables, cu = _attention_case(n, lens, [1] * 3, h, hk, dk, bs, F32)
    out = ops.kv8_attention(q.to(dev()), *[x.to(dev()) for x in cache], tables.to(dev()), _i32(lens)).cpu()
    for b, m in enumerate(lens):
        blocks = tables[b, :-(-m // bs)].long()
        for g in range(hk):
            k = (cache[0][blocks, g].double() * cache[2][blocks, g].double()[:, None, None]).reshape(-1, cache[0].shape[3])[:m, :dk]
            v = (cache[1][blocks, g].double() * cache[3][blocks, g].double()[:, None, None]).transpose(1, 2).reshape(-1, cache[0].shape[3])[:m, :dk]
            heads = slice(g * (h // hk), (g + 1) * (h // hk))
            p = torch.softmax(q[b, heads].double() @ k.t() / math.sqrt(dk), -1)
            want, spread = p @ v, p @ v.abs()
            err = (out[b, heads].double() - want).abs() - _bound(F32, q, cache, spread, want, 1 / math.sqrt(dk))
            assert bool((err <= 0).all()), (b, g, float(err.max()))


def _dense_reference(q, cache, tables, lens, cu, causal, scale):
    """(out, spread) in 64 bits on the GPU, sequence by sequence and head by head."""
    n, h, dk = q.shape
    hk, bs, w = cache[0].shape[1:]
    put = [t.to(dev()) for t in (q, *cache)]
    q, kc, vc, ks, vs = put
    out, spread = torch.zeros(n, h, dk, dtype=torch.float64, device=dev()), torch.zeros(n, h, dk, dtype=torch.float64, device=dev())
    for b, m in enumerate(lens):
        blocks = tables[b, :-(-m // bs)].long().to(dev())
        lo, hi = cu[b], cu[b + 1]
        place = m - (hi - lo) + torch.arange(hi - lo, device=dev()) if causal else torch.full((hi - lo,), m - 1, device=dev())
        hidden = torch.arange(m, device=dev())[None] > place[:, None]
        for i in range(h):
            g = i // (h // hk)
            k = (kc[blocks, g].double() * ks[blocks, g].double()[:, None, None]).reshape(-1, w)[:m, :dk]
            v = (vc[blocks, g].double() * vs[blocks, g].double()[:, None, None]).transpose(1, 2).reshape(-1, w)[:m, :dk]
            p = torch.softmax((q[lo:hi, i].double() @ k.t() * scale).masked_fill(hidden, -math.inf), -1)
            out[lo:hi, i], spread[lo:hi, i] = p @ v, p @ v.abs()
    return out.cpu(), spread.cpu()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("h,hk,dk,bs,lens,rows", [
    (8, 2, 128, 64, [3001, 700], [301, 130]),               # rows by the hundreds, the key axis split there too
    (4, 4, 64, 16, [1500, 1201, 65], [1500, 66, 65]),
    (6, 1, 24, 32, [900, 2500], [11, 200]),
    (8, 2, 128, 128, [5000, 40, 2300, 1], [1, 40, 300, 1]),  # single rows beside chunks
    (40, 1, 80, 16, [2100, 2100], [1, 9])])                 # one kv head for forty: a single token is forty rows
def test_attention_of_hundreds_of_rows(dtype, causal, h, hk, dk, bs, lens, rows):
    q, cache, tables, cu = _attention_case(sum(lens), lens, rows, h, hk, dk, bs, dtype)
    got = ops.kv8_attention(q.to(dev()), *[x.to(dev()) for x in cache], tables.to(dev()), _i32(lens), cu_rows=_i32(cu),
                            max_rows=max(rows), causal=causal).cpu().double()
    want, spread = _dense_reference(q, cache, tables, lens, cu, causal, 1 / math.sqrt(dk))
    err = (got - want).abs() - _bound(dtype, q, cache, spread, want, 1 / math.sqrt(dk))
    assert bool((err <= 0).all()), float(err.max())


def test_attention_offsets_beyond_32_bits():
    """A pool of more than 2^32 bytes: blocks at its far end."""
    nb, hk, bs, w = 4 * 1024 + 8, 16, 128, 128              # 1.05 GiB of codes each for 4104 blocks ...
    nb *= 5                                                 # ... 5 GiB
    kc = torch.zeros(nb, hk, bs, w, dtype=torch.int8, device=dev())
    vc = torch.zeros(nb, hk, w, bs, dtype=torch.int8, device=dev())
    ks, vs = torch.zeros(nb, hk, device=dev()), torch.zeros(nb, hk, device=dev())
    g = torch.Generator().manual_seed(3)
    last = nb - 1
    slots = [last * bs + i for i in range(20)] + [(last - 7) * bs + i for i in range(3)]
    k, v = (torch.randn(23, hk, w, generator=g) for _ in range(2))
    ops.kv8_append(k.to(dev()), v.to(dev()), _i32(slots), kc, vc, ks, vs)
    assert int((kc[:last - 8].view(-1)[::4097] != 0).sum()) == 0
    tables = torch.tensor([[last], [last - 7]], dtype=torch.int32)
    q = torch.randn(2, hk, w, generator=g)
    out = ops.kv8_attention(q.to(dev()), kc, vc, ks, vs, tables.to(dev()), _i32([20, 3])).cpu().double()
    small = [t[[last, last - 7]].cpu() for t in (kc, vc, ks, vs)]
    want, _, spread = ok.attention(q, *small, torch.tensor([[0], [1]], dtype=torch.int32), [20, 3], None, True, 1 / math.sqrt(w))
    assert bool(((out - want).abs() <= _bound(F32, q, small, spread, want, 1 / math.sqrt(w))).all())


# ------------------------------------------------------------------------------------------ logits
def _logits_case(seed, R, V, L, nb, dtype):
    g = torch.Generator().manual_seed(seed)
    x = (3 * torch.randn(R, V, generator=g)).to(dtype)
    kw = dict(history=torch.randint(-2, V + 2, (R, L), generator=g).to(torch.int32),
              history_len=torch.randint(0, L + 1, (R,), generator=g).to(torch.int32),
              repetition=1 + torch.rand(R, generator=g), presence=torch.rand(R, generator=g), frequency=torch.rand(R, generator=g))
    if L > 3:
        kw["history"][:, 1::2] = kw["history"][:, :1]        # one id over and over
    if nb:
        ids = torch.randint(-1, V + 1, (R, nb), generator=g).to(torch.int32)
        ids[:, nb // 2:] = ids[:, :nb - nb // 2]             # entries of one class twice
        kw.update(bias_ids=ids, bias_values=torch.randn(R, nb, generator=g))
    kw["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (R, (V + 31) // 32), generator=g).to(torch.int32)
    kw["bias"] = torch.randn(R, V, generator=g)
    return x, kw


def _check_logits(x, kw, out=None):
    put = lambda t: t.to(dev()) if t is not None else None
    got = ops.logits_process(put(x), **{k: put(t) for k, t in kw.items()}, **({} if out is None else dict(out=out)))
    want = ok.logits(x, **kw)
    g = got.double().cpu()
    assert torch.equal(torch.isneginf(g), torch.isneginf(want)) and torch.equal(torch.isnan(g), torch.isnan(want))
    fine = torch.isfinite(want)
    # at most 6 roundings in fp32 of intermediates below the sum of magnitudes, and one to the result's type
    n = kw["history"].shape[1] if kw.get("history") is not None else 0
    size = 2 * x.double().abs() + n + 2 + (kw["bias"].abs().max() if kw.get("bias") is not None else 0) + \
        (kw["bias_values"].abs().sum(-1).max() if kw.get("bias_values") is not None else 0)
    tol = torch.finfo(x.dtype).eps / 2 * want.abs() + 6 * 2.0 ** -24 * size
    assert bool(((g - want).abs()[fine] <= tol[fine]).all())
    return got


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("R,V,L,nb", [(1, 1, 1, 1), (3, 7, 5, 4), (2, 33, 40, 0), (10, 4233, 61, 8), (4, 8192, 300, 20),
                                      (3, 20001, 700, 300), (2, 8200, 3, 2), (2, 150, 9, 700)])
def test_logits(dtype, R, V, L, nb):
    x, kw = _logits_case(V, R, V, L, nb, dtype)
    _check_logits(x, kw)


@pytest.mark.parametrize("drop", ["history_len", "repetition", "presence", "frequency", "bias", "allowed", "biases", "penalties", "all"])
def test_logits_parts_may_be_left_out(drop):
    x, kw = _logits_case(1, 3, 500, 20, 6, F32)
    gone = {"biases": ["bias_ids", "bias_values"], "penalties": ["history", "history_len", "repetition", "presence", "frequency"],
            "all": list(kw)}.get(drop, [drop])
    for name in gone:
        del kw[name]
    got = _check_logits(x, kw)
    if drop == "all":
        assert torch.equal(got.cpu(), x)


def test_logits_shared_rows_padded_rows_and_in_place():
    x, kw = _logits_case(2, 4, 1000, 20, 6, F32)
    kw["bias"], kw["allowed"] = kw["bias"][:1], kw["allowed"][0]
    kw["bias_ids"], kw["bias_values"] = kw["bias_ids"][0], kw["bias_values"][:1]
    _check_logits(x, kw)
    wide = torch.zeros(4, 1008, device=dev())
    wide[:, :1000] = x.to(dev())
    rows = wide[:, :1000]
    put = {k: t.to(dev()) for k, t in kw.items()}
    want = ops.logits_process(x.to(dev()), **put)
    got = ops.logits_process(rows, **put, out=rows)
    assert got.data_ptr() == wide.data_ptr() and torch.equal(wide[:, :1000], want) and bool((wide[:, 1000:] == 0).all())


def test_logits_nothing_allowed_and_not_finite_logits():
    x = torch.tensor([[1.0, math.nan, math.inf, -math.inf], [math.nan, 2.0, -3.0, 4.0]])
    kw = dict(history=torch.tensor([[0, 1, 2, 3], [0, 2, 2, 2]], dtype=torch.int32), repetition=torch.tensor([2.0, 2.0]),
              presence=torch.tensor([0.5, 0.5]), allowed=torch.tensor([[0], [0b1100]], dtype=torch.int32))
    got = _check_logits(x, kw).cpu()
    assert bool((got[0] == -math.inf).all()) and got[1].tolist()[:2] == [-math.inf, -math.inf]
    del kw["allowed"]
    got = _check_logits(x, kw).cpu()
    assert math.isnan(got[0, 1]) and got[0, 2] == math.inf and got[0, 3] == -math.inf and got[1, 2] == -6.5


# ------------------------------------------------------------------------------------------ together
def test_streams_and_graphs():
    """A decoding step recorded once and replayed, with its own state moving on in place, equals eager steps."""
    hk, h, dk, bs, V, B = 2, 4, 64, 16, 300, 3
    g = torch.Generator().manual_seed(11)
    wq, wk, wv = (torch.randn(V, n, dk, generator=g).to(BF16).to(dev()) for n in (h, hk, hk))
    wo = torch.randn(h * dk, V, generator=g).to(dev()) / 8

    def fresh():
        s = dict(lens=_i32([0, 17, 40]), tables=torch.full((B, 8), -1, dtype=torch.int32, device=dev()), free=_i32(list(range(19, -1, -1))),
                 count=_i32([20]), token=_i32([5, 6, 7]), ones=_i32([1, 1, 1]), history=torch.zeros(B, 64, dtype=torch.int32, device=dev()),
                 hlen=_i32([0, 0, 0]), cache=[t.to(dev()) for t in _random_cache(torch.Generator().manual_seed(12), 20, hk, bs, 64, dk)],
                 rep=torch.full((B,), 1.3, device=dev()), logits=torch.zeros(B, V, device=dev()))
        prefill = _i32([0, 17, 40])
        zero = _i32([0, 0, 0])
        p = ops.kv_plan(zero, prefill, s["tables"], s["free"], s["count"], bs, 57)
        ids = torch.arange(57, device=dev()) % V
        ops.kv8_append(wk[ids], wv[ids], p.slots, *s["cache"])
        return s

    def step(s):
        p = ops.kv_plan(s["lens"], s["ones"], s["tables"], s["free"], s["count"], bs, B)
        t = s["token"].long()
        ops.kv8_append(wk[t], wv[t], p.slots, *s["cache"])
        o = ops.kv8_attention(wq[t], *s["cache"], s["tables"], s["lens"])
        x = ops.logits_process(o.float().view(B, -1) @ wo, history=s["history"], history_len=s["hlen"], repetition=s["rep"])
        s["logits"].copy_(x)
        s["token"].copy_(x.argmax(-1))
        s["history"].scatter_(1, s["hlen"][:, None].long(), s["token"][:, None])
        s["hlen"].add_(1)

    eager = fresh()
    want = []
    for _ in range(20):
        step(eager)
        want.append((eager["logits"].clone(), eager["token"].tolist()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = fresh()
        step(warm)
        got = fresh()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(got)
    for i in range(20):
        graph.replay()
        torch.cuda.synchronize()
        step(warm)                                          # the program's own eager work in between
        assert torch.equal(got["logits"], want[i][0]) and got["token"].tolist() == want[i][1], i
    assert torch.equal(got["tables"], eager["tables"]) and int(got["count"]) == int(eager["count"])


def test_two_streams_at_once_give_the_same():
    lens, rows = [5000, 3000], [1, 1]
    q, cache, tables, cu = _attention_case(13, lens, rows, 8, 2, 128, 64, BF16)
    args = [x.to(dev()) for x in (q, *cache, tables)] + [_i32(lens)]
    want = ops.kv8_attention(*args)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(ops.kv8_attention(*args))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


# ------------------------------------------------------------------------------------------ odd calls
@pytest.mark.parametrize("places", [[5, 4, 4, 7], [3, 3, 3], [9, 0, 15], [15, 14, 13, 12, 11, 10], [6, -1, 7, -1, -1, 8]])
def test_append_rows_out_of_order_twice_and_with_gaps(places):
    g = torch.Generator().manual_seed(len(places))
    other = [32 + i for i in range(5)]                      # another block before and behind
    slots = other[:2] + [16 + p if p >= 0 else -1 for p in places] + [48, 49] + [-1] * 300
    k, v = (torch.randn(len(slots), 2, 40, generator=g).to(BF16) for _ in range(2))
    got, want = _append_both(k, v, slots, _random_cache(g, 4, 2, 16, 64, 40))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_append_a_run_far_behind_skipped_rows():
    g = torch.Generator().manual_seed(1)
    slots = [16, 17] + [-1] * 700 + [18, 19] + [-1] * 130 + [20, 40]
    k, v = (torch.randn(len(slots), 1, 32, generator=g) for _ in range(2))
    got, want = _append_both(k, v, slots, _random_cache(g, 4, 1, 16, 32, 32))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("shift", [0, 1, 3])
def test_append_of_rows_that_do_not_lie_on_pairs(shift):
    g = torch.Generator().manual_seed(shift)
    slots = list(range(3, 40))
    k, v = (torch.randn(37, 2, 67, generator=g).to(BF16).to(dev())[..., shift:shift + 33] for _ in range(2))
    got, want = _append_both(k, v, slots, _random_cache(g, 4, 2, 16, 64, 33))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_append_of_broadcast_rows():
    g = torch.Generator().manual_seed(2)
    one = torch.randn(1, 1, 32, generator=g).to(dev()).expand(20, 2, 32)
    got, want = _append_both(one, -one, list(range(20)), _random_cache(g, 2, 2, 16, 32, 32))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_attention_with_a_negative_scale_and_results_over_the_queries():
    lens = [70, 33]
    q, cache, tables, cu = _attention_case(21, lens, [1, 1], 4, 2, 64, 16, F32)
    _check_attention(q, cache, tables, lens, cu, True, F32, scale=-0.2, one_row=True)
    _check_attention(q, cache, tables, lens, cu, True, F32, scale=0.0, one_row=True)
    args = [x.to(dev()) for x in (q, *cache, tables)] + [_i32(lens)]
    want = ops.kv8_attention(*args)
    got = ops.kv8_attention(*args, out=args[0])
    assert got.data_ptr() == args[0].data_ptr() and torch.equal(got, want)


def test_a_split_attention_in_two_graphs():
    """Each recorded call has a workspace of its own: replays in turn, with eager calls between them."""
    lens = [5000, 2500]
    cases = [_attention_case(s, lens, [1, 1], 8, 2, 128, 64, BF16) for s in (31, 32)]
    args = [[x.to(dev()) for x in (q, *cache, tables)] + [_i32(lens)] for q, cache, tables, _ in cases]
    want = [ops.kv8_attention(*a) for a in args]
    assert not torch.equal(*want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    for a in args:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(ops.kv8_attention(*a))
        graphs.append(g)
    for i in range(6):
        for o in outs:
            o.zero_()
        for j in ((0, 1), (1, 0))[i % 2]:
            graphs[j].replay()
        assert torch.equal(ops.kv8_attention(*args[i % 2]), want[i % 2])
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want)), i


def test_tensors_elsewhere_are_refused():
    lens = [20]
    q, cache, tables, cu = _attention_case(22, lens, [1], 2, 2, 64, 16, F32)
    put = [x.to(dev()) for x in (q, *cache, tables)] + [_i32(lens)]
    for i in range(len(put)):
        mixed = list(put)
        mixed[i] = mixed[i].cpu()
        with pytest.raises(RuntimeError, match="current GPU"):
            ops.kv8_attention(*mixed)
    with pytest.raises(RuntimeError, match="current GPU"):
        ops.kv8_append(q, put[0], _i32([0]), *put[1:5])
    with pytest.raises(RuntimeError, match="current GPU"):
        ops.logits_process(torch.zeros(2, 40), history=_i32([[1], [2]]))
    same = _i32([1, 2])
    with pytest.raises(RuntimeError, match="new_rows"):
        ops.kv_plan(same, same, torch.zeros(2, 4, dtype=torch.int32, device=dev()), _i32([1]), _i32([1]), 16, 3)
    with pytest.raises(TypeError, match="dtype"):
        ops.kv8_attention(put[0].half(), *put[1:])


@pytest.mark.parametrize("width", [1, 60, 61, 62, 63, 64, 65, 127, 128])
def test_attention_with_tables_around_the_first_split(width):
    """Tables of 16 .. 2048 places: the key axis is first divided at 1024."""
    lens = [16 * width, 5]
    q, cache, tables, cu = _attention_case(width, lens, [1, 1], 2, 1, 32, 16, F32)
    assert tables.shape[1] == width
    got = ops.kv8_attention(q.to(dev()), *[x.to(dev()) for x in cache], tables.to(dev()), _i32(lens)).cpu().double()
    want, spread = _dense_reference(q, cache, tables, lens, cu, True, 1 / math.sqrt(32))
    assert bool(((got - want).abs() <= _bound(F32, q, cache, spread, want, 1 / math.sqrt(32))).all())


# ------------------------------------------------------------------------------------------ one key far above the others
def _far_case(seed, lens, rows, h, hk, dk, bs, dtype, top, amp, ks, dominant_value=None):
    """Every sequence's first token stands ``top`` (in natural units, over scores of deviation ``amp``) above the others: queries are one number
    throughout and the first key's codes add up to it, so that sums over columns are whole numbers times a power of two and exact in fp32."""
    q, cache, tables, cu = _attention_case(seed, lens, rows, h, hk, dk, bs, dtype)
    kc, vc, k_scale, v_scale = cache
    g = torch.Generator().manual_seed(seed + 1)
    scale = 1 / math.sqrt(dk)
    # deviation of a sum of dk codes of -n .. n: sqrt(dk n (n + 1) / 3)
    n = 20
    c = 2.0 ** round(math.log2(amp / (scale * ks * math.sqrt(dk * n * (n + 1) / 3))))
    q[:] = c
    kc[..., :dk] = torch.randint(-n, n + 1, kc[..., :dk].shape, generator=g, dtype=torch.int8)
    k_scale[:] = ks
    total = round(top / (c * ks * scale))
    assert abs(total) <= 127 * dk
    first = [int(tables[b, 0]) for b in range(len(lens))]
    for j in range(dk):
        kc[first, :, 0, j] = (total + j) // dk              # (adds up to ``total``)
    if dominant_value is not None:
        vc[first, :, :dk, 0] = dominant_value
    return q, cache, tables, cu, scale


# (sequences, rows, heads): single rows, whole and split key axis; a few rows; rows by the hundreds, whole and split
FAR_SHAPES = [([64, 1000, 700], [1, 1, 1], 4, 2, 64, 16), ([20000, 64], [1, 1], 8, 2, 128, 64), ([640, 300], [5, 9], 4, 2, 32, 16),
              ([500, 260], [300, 200], 4, 4, 64, 32), ([4001, 1000], [300, 70], 8, 2, 128, 64)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lens,rows,h,hk,dk,bs", FAR_SHAPES)
@pytest.mark.parametrize("which", ["all", "first"])
def test_attention_value_scales_of_zero_beside_large_scores(dtype, lens, rows, h, hk, dk, bs, which):
    """Blocks of zeros have scale 0; a score of 120 above the others (173 in units of two) must not turn them into NaN.  Where the first key's
    block is such a block the others' share is e^-120 and less: zero in fp32."""
    q, cache, tables, cu, scale = _far_case(5, lens, rows, h, hk, dk, bs, dtype, 120.0, 3.0, 0.5)
    if which == "all":
        cache[3][:] = 0
    else:
        cache[3][[int(tables[b, 0]) for b in range(len(lens))]] = 0
    one_row = max(rows) == 1
    for causal in (True, False):
        got = ops.kv8_attention(q.to(dev()), *[x.to(dev()) for x in cache], tables.to(dev()), _i32(lens), cu_rows=None if one_row else _i32(cu),
                                max_rows=max(rows), causal=causal, scale=scale)
        assert bool((got.double().abs() < 1e-37).all()), float(got.double().abs().max())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lens,rows,h,hk,dk,bs", FAR_SHAPES)
@pytest.mark.parametrize("top", [50.0, 1000.0, 2e4, 1e6, 3e7])
def test_attention_one_key_takes_everything_in_whole_tiles(dtype, lens, rows, h, hk, dk, bs, top):
    """The result is that key's value: two roundings of a product (2^-22 / 2^-11), whatever the size of the scores."""
    q, cache, tables, cu, scale = _far_case(6, lens, rows, h, hk, dk, bs, dtype, top, top / 50, top / 1024)
    got = ops.kv8_attention(q.to(dev()), *[x.to(dev()) for x in cache], tables.to(dev()), _i32(lens), cu_rows=None if max(rows) == 1 else _i32(cu),
                            max_rows=max(rows), causal=True, scale=scale).cpu().double()
    first = tables[:, 0].long()
    value = (cache[1][first][..., :dk, 0].double() * cache[3][first].double()[..., None]).repeat_interleave(h // hk, 1)
    want = torch.cat([value[b:b + 1].expand(r, -1, -1) for b, r in enumerate(rows)])
    tol = (torch.finfo(dtype).eps / 2 + (2.0 ** -11 if dtype == BF16 else 2.0 ** -20)) * want.abs()
    # (at 50 the others' share is e^-45 of some thousands)
    assert bool(((got - want).abs() <= tol + 1e-14).all()), float(((got - want).abs() / want.abs().clamp(min=1e-30)).max())


def _check_far(q, cache, tables, lens, cu, dtype, scale, causal, one_row, top):
    """What is left of the bound where the sums of the scores are exact: the exponent's four roundings (the score's factor twice, the running
    maximum, the difference), each 2^-24 of the score in units of two (1.45 top); probabilities as in ``_bound``; and products below 2^-40 of the
    row's largest, which vanish."""
    got = ops.kv8_attention(q.to(dev()), *[x.to(dev()) for x in cache], tables.to(dev()), _i32(lens), cu_rows=None if one_row else _i32(cu),
                            max_rows=max(b - a for a, b in zip(cu, cu[1:])), causal=causal, scale=scale).cpu().double()
    want, spread = _dense_reference(q, cache, tables, lens, cu, causal, scale)
    inner = 4 * 2.0 ** -24 * 1.45 * (top + 4) + (2.0 ** -11 if dtype == BF16 else 2.0 ** -20)
    vmax = float((cache[1].float().abs().amax((1, 2, 3)) * cache[3].amax(1)).max())
    err = (got - want).abs() - torch.finfo(dtype).eps / 2 * want.abs() - inner * spread - max(lens) * 2.0 ** -40 * vmax
    assert bool((err <= 0).all()), (float(err.max()), float(((got - want).abs() / (inner * spread + 1e-300)).max()))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lens,rows,h,hk,dk,bs", FAR_SHAPES)
@pytest.mark.parametrize("top", [8.0, 10.0, 12.0, 14.0, 16.0])
def test_attention_beside_a_key_that_dominates(dtype, lens, rows, h, hk, dk, bs, top):
    """A first token that takes most of the mass and whose value is nothing: the result is what the others, e^-top each, come to."""
    case = _far_case(int(top), lens, rows, h, hk, dk, bs, dtype, top, 0.5, 1 / 16, dominant_value=0)
    for causal in (True, False):
        _check_far(*case[:3], lens, case[3], dtype, case[4], causal, max(rows) == 1, top)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("below", [24.5, 25.1, 28.0])
def test_attention_of_a_long_flat_tail(dtype, below):
    """131071 equal tokens 2^-24.5 and less of the first one's weight each: 0.55 % to 0.05 % of the result together."""
    q, cache, tables, cu, scale = _far_case(3, [131072], [1], 2, 1, 64, 64, dtype, below * math.log(2), 0.5, 1 / 16, dominant_value=100)
    cache[0].zero_()                                        # every code 0 ...
    first = int(tables[0, 0])
    total = round(below * math.log(2) / (float(q[0, 0, 0]) / 16 * scale))
    for j in range(64):
        cache[0][first, :, 0, j] = (total + j) // 64        # ... but the first key's
    cache[1][..., :64, :] = 90
    cache[1][first, :, :64, 0] = 0
    cache[3][:] = 0.013
    _check_far(q, cache, tables, [131072], cu, dtype, scale, True, True, below * math.log(2))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lens,rows,h,hk,dk,bs", FAR_SHAPES)
@pytest.mark.parametrize("small", [-14, -20, -24])
def test_attention_queries_with_columns_of_very_different_sizes(dtype, lens, rows, h, hk, dk, bs, small):
    """Scores made of columns 2^-14 and less of the row's largest, whose keys are zero.  A column is held to 2^-22 of itself (fp32; bf16
    queries exactly) or 2^-39 of the largest; the rest as in ``_bound``."""
    q, cache, tables, cu = _attention_case(11, lens, rows, h, hk, dk, bs, dtype)
    q[..., 1:] = (q[..., 1:].float() * 2.0 ** small).to(dtype)
    q[..., 0] = 1.5
    cache[0][..., 0] = 0
    cache[2][:] *= 2.0 ** -small
    scale = 1 / math.sqrt(dk)
    got = ops.kv8_attention(q.to(dev()), *[x.to(dev()) for x in cache], tables.to(dev()), _i32(lens), cu_rows=None if max(rows) == 1 else _i32(cu),
                            max_rows=max(rows), causal=True, scale=scale).cpu().double()
    want, spread = _dense_reference(q, cache, tables, lens, cu, True, scale)
    kmax = 127 * float(cache[2].max())
    x = q.double().abs()
    x[..., 0] = 0
    held = torch.maximum(2.0 ** -22 * x, torch.tensor(2.0 ** -39 * 2).double()).sum(-1).max() if dtype == F32 else 2.0 ** -39 * 2 * dk
    score = kmax * scale * (6 * math.sqrt(dk + 8) * 2.0 ** -24 * float(x.sum(-1).max()) + float(held))
    inner = 2 * score + (2.0 ** -11 if dtype == BF16 else 2.0 ** -20)
    err = (got - want).abs() - torch.finfo(dtype).eps / 2 * want.abs() - inner * spread
    assert bool((err <= 0).all()), (float(err.max()), float(((got - want).abs() / (inner * spread)).max()))


def test_append_a_run_of_very_many_skipped_rows():
    """2^24 skipped rows inside a run of heads of 128: rows times columns pass 2^31."""
    g = torch.Generator().manual_seed(3)
    one = torch.randn(1, 1, 128, generator=g).to(BF16)
    n = 2 ** 24 + 3
    slots = torch.full((n,), -1, dtype=torch.int32, device=dev())
    slots[0], slots[n - 2], slots[n - 1] = 18, 19, 40
    cache = _random_cache(g, 4, 1, 16, 128, 128)
    got = [t.to(dev()) for t in cache]
    rows = one.to(dev()).expand(n, 1, 128)
    ops.kv8_append(rows, -rows, slots, *got)
    few, want = one.expand(3, 1, 128), [t.clone() for t in cache]
    ok.append(few, [18, 19, 40], want[0], want[2])
    vt = want[1].transpose(2, 3).contiguous()
    ok.append(-few, [18, 19, 40], vt, want[3])
    want[1] = vt.transpose(2, 3)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))


@pytest.mark.parametrize("N", [512, 513, 2047, 2048, 2049, 2200])
def test_append_rows_of_every_workgroup_size(N):
    """2048 and 8192 rows x heads are where the rows of a workgroup change (4 heads): single rows, short runs, long ones, gaps."""
    g = torch.Generator().manual_seed(N)
    bs, hk, dk = 16, 4, 32
    blocks = torch.randperm(N // 2 + 400, generator=g).tolist()
    slots, at = [], 0
    while len(slots) < N:
        kind = at % 4
        first, n = [(at % bs, 1), (3, 9), (0, 40), (15, 2)][kind]
        for j in range(n):
            slots.append(blocks[at + (first + j) // bs] * bs + (first + j) % bs)
        if kind == 1:
            slots += [-1] * (at % 3)
        at += (first + n - 1) // bs + 1
    slots = slots[:N]
    k, v = (torch.randn(N, hk, dk, generator=g).to(BF16) for _ in range(2))
    got, want = _append_both(k, v, slots, _random_cache(g, len(blocks), hk, bs, 32, dk))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("top", [-700.0, -100.0, 300.0, 700.0])
@pytest.mark.parametrize("lens,rows,h,hk,dk,bs", FAR_SHAPES)
def test_attention_of_large_scores_in_one_exponential(lens, rows, h, hk, dk, bs, top):
    """bf16 below 1024 in units of two, where a score and a value scale's logarithm meet in one number: twice 2^-14 of an exponent is 8.5e-5
    of a term, within the 2^-11 of ``_bound``; so are scores that are all far below 0 (one key above the others takes everything).  Products
    below 2^-40 of the row's largest vanish, as in ``_check_far``: where the first value is 0, what is left are the others', e^-100 and less."""
    q, cache, tables, cu, scale = _far_case(8, lens, rows, h, hk, dk, bs, BF16, abs(top), abs(top) / 50, abs(top) / 1024)
    if top < 0:
        cache[0][..., :dk] = (cache[0][..., :dk].int() // 16 - 40).to(torch.int8)
        first = [int(tables[b, 0]) for b in range(len(lens))]
        cache[0][first, :, 0, :dk] = -30
    got = ops.kv8_attention(q.to(dev()), *[x.to(dev()) for x in cache], tables.to(dev()), _i32(lens), cu_rows=None if max(rows) == 1 else _i32(cu),
                            max_rows=max(rows), causal=True, scale=scale).cpu().double()
    want, spread = _dense_reference(q, cache, tables, lens, cu, True, scale)
    vmax = float((cache[1].float().abs().amax((1, 2, 3)) * cache[3].amax(1)).max())
    tol = _bound(BF16, q, cache, spread, want, scale) + max(lens) * 2.0 ** -40 * vmax
    assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() / tol.clamp(min=1e-30)).max())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("which", [2, 3])
@pytest.mark.parametrize("lens,rows,h,hk,dk,bs", FAR_SHAPES)
def test_attention_scales_that_are_not_finite_in_whole_tiles(dtype, which, lens, rows, h, hk, dk, bs):
    """Rows that see such a block are NaN, those in front of it and the other kv heads are what they were, to the bit."""
    q, cache, tables, cu = _attention_case(14, lens, rows, h, hk, dk, bs, dtype)
    call = lambda: ops.kv8_attention(q.to(dev()), *[x.to(dev()) for x in cache], tables.to(dev()), _i32(lens),
                                     cu_rows=None if max(rows) == 1 else _i32(cu), max_rows=max(rows)).cpu()
    want = call()
    hit = [(n - r // 2 - 1) // bs for n, r in zip(lens, rows)]
    for b, j in enumerate(hit):
        cache[which][int(tables[b, j]), hk - 1] = math.nan
    got = call()
    for b, (n, r) in enumerate(zip(lens, rows)):
        sees = torch.arange(n - r, n) >= hit[b] * bs
        nan = torch.zeros(r, h, dtype=torch.bool)
        nan[sees, h - h // hk:] = True
        part = got[cu[b]:cu[b + 1]]
        assert torch.equal(torch.isnan(part).any(-1), nan) and torch.equal(torch.isnan(part).all(-1), nan)
        assert torch.equal(part[~nan], want[cu[b]:cu[b + 1]][~nan])
