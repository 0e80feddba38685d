"""Attention over router-chosen blocks at its borders: sizes, layouts, memory and values that ordinary calls do not reach."""
from __future__ import annotations

import math

import pytest
import torch

import block_attention_util as plain
from relation_lm.kernels import block_attention as ba

pytestmark = pytest.mark.gpu

DTYPES = (torch.float32, torch.bfloat16, torch.float16)
HALF_TYPES = (torch.bfloat16, torch.float16)


def random(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def within(got, want, bound, what=""):
    error = (got.double().cpu() - want).abs()
    assert bool((error <= bound).all()), (what, float((error - bound).max()))


def status_clear():
    from relation_lm.kernels import _abi

    assert _abi.read_status() == 0


def check_rows(some, at, q, k_cache, v_cache, index, out, lse, block_size, window, scale):
    """Rows ``some`` of a call against the 64-bit form; ``index`` is [rows, kv_heads, places]."""
    for i in some:
        b, t = at[i]
        want, want_lse, bound, lse_bound = plain.attend(q[i].cpu(), k_cache[b].cpu(), v_cache[b].cpu(), index[i].cpu(), t, block_size,
                                                        window, scale)
        within(out[i], want, bound, (i, b, t))
        empty = want_lse == -math.inf
        assert bool((lse[i].cpu()[empty] == -math.inf).all())
        within(lse[i].cpu()[~empty], want_lse[~empty], lse_bound[~empty], "lse")


# ---------------------------------------------------------------------------- blocks longer than the cache


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form", ("decode", "rows", "prefill"))
@pytest.mark.parametrize("context,window", [(9, 2), (200, 30)])
@pytest.mark.parametrize("block_size", ("one more", 1 << 20, "most"))
def test_blocks_longer_than_the_cache(dtype, form, context, window, block_size):
    # the first block is then all that lies before the window; the largest size that the entry point takes among them
    block_size = {"one more": context + 1, "most": 0x7fffffff - context}.get(block_size, block_size)
    g = torch.Generator().manual_seed(context)
    at = [(b, context - 1) for b in range(2)] if form == "decode" else plain.places(form, 2, min(2 * context, 25), context, context)
    n = len(at)
    q = random(g, n, 4, 64, dtype=dtype)
    k_cache, v_cache = (random(g, 2, context, 2, 64, dtype=dtype) for _ in range(2))
    index = torch.tensor([0, 1, 0, -1], dtype=torch.int32).expand(n, 2, 4)
    call = {"decode": ba.block_attention, "rows": ba.block_attention_rows, "prefill": ba.block_attention_prefill}[form]
    out, lse = call(q.cuda(), k_cache.cuda(), v_cache.cuda(), index.cuda(), *plain.where(form, at, context), block_size, window, 0.125)
    check_rows(range(0, n, 1 + n // 40), at, q, k_cache, v_cache, index, out, lse, block_size, window, 0.125)
    status_clear()


@pytest.mark.parametrize("dtype", HALF_TYPES)
@pytest.mark.parametrize("width", (64, 96))
@pytest.mark.parametrize("block_size,spare", [(500, 0), (601, 0), (1 << 20, 70), (0x7fffffff - 671, 70)])
def test_blocks_longer_than_whole_sequences(dtype, width, block_size, spare):
    length, window = 601, 40
    g = torch.Generator().manual_seed(width)
    at = plain.places("prefill", 2, 0, 0, length)
    q = random(g, len(at), 4, width, dtype=dtype)
    k_cache, v_cache = (random(g, 2, length + spare, 2, width, dtype=dtype) for _ in range(2))
    k_cache[:, length:], v_cache[:, length:] = math.nan, math.inf            # nothing has been written there yet
    index = torch.randint(-1, 3, (len(at), 2, 3), generator=g, dtype=torch.int32)
    out, lse = ba.block_attention_prefill(q.cuda(), k_cache.cuda(), v_cache.cuda(), index.cuda(), length, block_size, window, 0.125)
    check_rows([0, 1, window, 300, 600, 601, 777, 1200, 1201], at, q, k_cache, v_cache, index, out, lse, block_size, window, 0.125)
    status_clear()


# ---------------------------------------------------------------------------- caches in one buffer


def _pairs_of_views():
    """(what, key cache, value cache, whether they have an element in common), [2, 6, 2, 32] each."""
    def buffer(*shape):
        return torch.randn(*shape, device="cuda").bfloat16()

    three, heads, wide = buffer(3, 6, 2, 32), buffer(2, 6, 3, 32), buffer(2, 6, 2, 48)
    long, apart, kv = buffer(2, 9, 2, 32), buffer(2, 12, 2, 32), buffer(2, 6, 2, 2, 32)
    return [("sequences", three[:2], three[1:], True),
            ("heads", heads[:, :, :2], heads[:, :, 1:], True),
            ("components", wide[..., :32], wide[..., 16:], True),
            ("positions", long[:, :6], long[:, 3:], True),
            ("orders", heads[:, :, :2], heads.view(2, 3, 6, 32)[:, 1:].transpose(1, 2), True),
            ("the same", three[:2], three[:2], True),
            ("every other position", apart[:, ::2], apart[:, 1::2], False),
            ("halves", apart[:, :6], apart[:, 6:], False),
            ("side by side", kv[:, :, 0], kv[:, :, 1], False),
            ("heads side by side", kv.view(2, 6, 4, 32)[:, :, :2], kv.view(2, 6, 4, 32)[:, :, 2:], False),
            ("components side by side", kv.view(2, 6, 2, 64)[..., :32], kv.view(2, 6, 2, 64)[..., 32:], False)]


@pytest.mark.parametrize("which", range(11))
def test_caches_that_overlap_are_refused(which):
    what, k_cache, v_cache, common = _pairs_of_views()[which]
    assert k_cache.shape == v_cache.shape == (2, 6, 2, 32)
    q, k, v = (torch.randn(2, n, 32, device="cuda").bfloat16() for n in (4, 2, 2))
    f, at = ba.rotary_frequencies(32, device="cuda")[0], torch.tensor(4, device="cuda")
    if common:
        with pytest.raises(ValueError, match="in common"):
            ba.rotary_append(q, k, v, k_cache, v_cache, f, at)
        with pytest.raises(ValueError, match="in common"):
            ba.rotary_append(q, k, v, v_cache, k_cache, f, at)
        return
    apart = k_cache.clone(), v_cache.clone()
    out, want = ba.rotary_append(q, k, v, k_cache, v_cache, f, at), ba.rotary_append(q, k, v, *apart, f, at)
    assert torch.equal(out, want) and torch.equal(k_cache, apart[0]) and torch.equal(v_cache, apart[1]), what


# ---------------------------------------------------------------------------- one row, one sequence, one head


@pytest.mark.parametrize("dtype", DTYPES)
def test_steps_that_lead_nowhere(dtype):
    # one row of a projection whose width is odd, caches of one sequence (or of one head) cut from buffers of odd widths
    g = torch.Generator().manual_seed(4)
    q = random(g, 2, 8 * 64 + 3, dtype=dtype).cuda()[:, :512].unflatten(1, (8, 64))[:1]
    caches = [random(g, 2, 40 * 128 + 5, dtype=dtype).cuda()[:, :40 * 128].unflatten(1, (40, 2, 64))[:1] for _ in range(2)]
    assert q.stride(0) % 2 == 1 and caches[0].stride(0) % 2 == 1
    index = torch.tensor([[[1, 0], [2, -1]]], dtype=torch.int32, device="cuda")
    at = torch.tensor(37, device="cuda")
    out, lse = ba.block_attention(q, *caches, index, at, 8, 6, 0.125)
    check_rows([0], [(0, 37)], q, *caches, index, out, lse, 8, 6, 0.125)
    one = [torch.as_strided(c, (1, 40, 1, 64), (c.stride(0), 128, 63, 1)) for c in caches]
    out, lse = ba.block_attention(q, *one, index[:, :1], at, 8, 6, 0.125)
    check_rows([0], [(0, 37)], q, *one, index[:, :1], out, lse, 8, 6, 0.125)
    # and into them
    k, v = (random(g, 2, 2 * 64 + 1, dtype=dtype).cuda()[:, :128].unflatten(1, (2, 64))[:1] for _ in range(2))
    f, plainly = ba.rotary_frequencies(64, device="cuda")[0], [c.clone(memory_format=torch.contiguous_format) for c in caches]
    turned = ba.rotary_append(q, k, v, *caches, f, at)
    assert torch.equal(turned, ba.rotary_append(q.contiguous(), k.contiguous(), v.contiguous(), *plainly, f, at))
    assert all(torch.equal(a, b) for a, b in zip(caches, plainly))
    within(turned, *plain.turned(q.cpu(), 37, f.cpu(), False, 1.0))
    status_clear()


# ---------------------------------------------------------------------------- values that are not finite, and neighbours


@pytest.mark.parametrize("dtype", HALF_TYPES)
@pytest.mark.parametrize("width,block_size", [(64, 16), (64, 64), (128, 32), (32, 16), (96, 64), (64, 100)])
def test_a_row_does_not_hang_on_its_neighbours(dtype, width, block_size):
    # every block ends in a value that is not finite.  Rows that see whole blocks stay as they are, to the last bit, whether or
    # not rows whose window begins within the same block choose it as well; and every call gives the same
    length, window, heads = 1500, 24, 4
    g = torch.Generator().manual_seed(width + block_size)
    q = random(g, length, heads, width, dtype=dtype).cuda()
    k_cache, v_cache = (random(g, 1, length, 2, width, dtype=dtype).cuda() for _ in range(2))
    v_cache[0, block_size - 1::block_size, :, 5] = math.inf
    t = torch.arange(length)
    start = (t - window + 1).clamp(min=0)
    whole = start // block_size                          # blocks that end before the window
    far = (torch.rand(length, generator=g) * whole).int()
    plain_rows = (t % 2 == 0) & (whole > 0)
    alone = torch.where(plain_rows, far, -1).int()
    beside = torch.where((t % 2 == 1) & (start % block_size > 0), start // block_size, alone).int()
    assert int((beside >= 0).sum()) > int((alone >= 0).sum()) + 400

    def call(index):
        return ba.block_attention_prefill(q, k_cache, v_cache, index[:, None].cuda(), length, block_size, window, 0.125)

    out, lse = call(alone)
    assert not bool(out[plain_rows.cuda()][..., 5].isfinite().any()) and bool(out[plain_rows.cuda()][..., 6:].isfinite().all())
    with_others, lse_with = call(beside)
    rest = torch.arange(width) != 5
    assert torch.equal(out[plain_rows.cuda()][..., rest], with_others[plain_rows.cuda()][..., rest])
    assert torch.equal(lse[plain_rows.cuda()], lse_with[plain_rows.cuda()])
    for _ in range(3):
        again, lse_again = call(beside)
        assert torch.equal(again.view(torch.int16), with_others.view(torch.int16)) and torch.equal(lse_again, lse_with)
    cpu = [x.cpu() for x in (q, k_cache, v_cache)]
    for i in range(200, length, 61):                     # the other components, against the 64-bit form
        finite = cpu[2].nan_to_num(posinf=0.0)
        want, want_lse, bound, lse_bound = plain.attend(cpu[0][i], cpu[1][0], finite[0], beside[i].expand(2, 1), i, block_size, window, 0.125)
        within(with_others[i][..., rest], want[..., rest], bound[..., rest], i)
        within(lse_with[i], want_lse, lse_bound)
    status_clear()


# ---------------------------------------------------------------------------- weights far below the largest


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form", ("decode", "rows", "prefill"))
@pytest.mark.parametrize("width,block_size", [(64, 64), (128, 32), (32, 16), (64, 100)])
def test_many_small_weights_count(dtype, form, width, block_size):
    # one key of every 50 outweighs each of the others 2^26-fold, but its value is zero and theirs are large: the result is
    # theirs.  Scores are whole powers of two, so that nothing but the rounding of the weights and of the result is left
    length, window, heads, top = 1300, 120, 4, 4          # whole sequences: as many rows as take the three passes
    g = torch.Generator().manual_seed(width)
    at = [(0, 897)] if form == "decode" else [(0, t) for t in range(700, 1300, 29)] if form == "rows" else plain.places(form, 1, 0, 0, length)
    n = len(at)
    q = torch.zeros(n, heads, width, dtype=dtype)
    q[..., 0] = 1.0
    k_cache = torch.zeros(1, length, 1, width, dtype=dtype)
    k_cache[0, ::50, 0, 0] = 26.0
    v_cache = (torch.rand(1, length, 1, width, generator=g) * 3.0e4 + 3.0e4).to(dtype)
    v_cache[0, ::50] = 0.0
    index = torch.randint(0, -(-length // block_size), (n, 1, top), generator=g, dtype=torch.int32)
    scale = math.log(2.0)
    call = {"decode": ba.block_attention, "rows": ba.block_attention_rows, "prefill": ba.block_attention_prefill}[form]
    out, lse = call(q.cuda(), k_cache.cuda(), v_cache.cuda(), index.cuda(), *plain.where(form, at, length), block_size, window, scale)
    step = plain.HALF_STEP[dtype]
    for i in range(0, n, 1 + n // 60):
        t = at[i][1]
        start = max(0, t - window + 1)
        keys = set(range(start, t + 1))
        for b in index[i, 0].tolist():
            keys |= set(range(b * block_size, min((b + 1) * block_size, start)))
        keys = sorted(keys)
        p = torch.exp2(k_cache[0, keys, 0, 0].double())
        want = (p @ v_cache[0, keys, 0].double()) / p.sum()
        # the scale times log2(e) in 32 bits: 2^-24 each and of the product, times 26 in the exponent and ln 2; powers (2 ulp),
        # sums over the keys; weights and the result rounded to the type, the latter to fp16's smallest steps
        weight = 2 * 3 * 2.0 ** -24 * 26 * math.log(2.0) + (len(keys) + 16) * 2.0 ** -24
        bound = (weight + (2 * step if dtype != torch.float32 else step)) * 1.01 * want + (2.0 ** -25 if dtype == torch.float16 else 0.0)
        within(out[i], want.expand(heads, width), bound.expand(heads, width), (i, t))
        within(lse[i], p.sum().log().expand(heads), torch.full((heads,), 1e-5, dtype=torch.float64))
    status_clear()


# ---------------------------------------------------------------------------- the choice, and the selectors beside it


def _statistics(g, batch, blocks, dtype=torch.float32):
    mean, std = random(g, batch, blocks, 4, 16, dtype=dtype, scale=0.5), random(g, batch, blocks, 4, 16, dtype=dtype, scale=0.5).abs()
    return mean, std, random(g, 4), random(g, 4, 9)


@pytest.mark.parametrize("place", [(2, 5), (-1, 5), (2, 0), (1 << 30, 1 << 30)])
def test_route_tells_each_row_outside_the_statistics(place):
    from relation_lm.kernels import _abi

    x = [v.cuda() for v in _statistics(torch.Generator().manual_seed(1), 2, 6)]
    q = torch.randn(1, 64, device="cuda")
    row = [torch.tensor([v], dtype=torch.int32, device="cuda") for v in place]
    index, score = ba.route_blocks_rows(q, *x, *row, 4, 2, 3, True)
    assert _abi.read_status() == 2 and index.tolist() == [[-1] * 3] and score.tolist() == [[-math.inf] * 3]
    index, score = ba.route_blocks(q.expand(2, 64).contiguous(), *x, torch.tensor(-1, device="cuda"), 4, 2, 3, True)
    assert _abi.read_status() == 2 and index.tolist() == [[-1] * 3] * 2


@pytest.mark.parametrize("blocks,block_size,top", [(2, 4, 1), (6, 4, 3), (700, 16, 40)])
@pytest.mark.parametrize("beyond", (0, 1, 1000, 0x7fffffff - 700 * 16 - 1))
def test_beyond_the_statistics_all_blocks_are_complete(blocks, block_size, top, beyond):
    g = torch.Generator().manual_seed(blocks)
    mean, std, gamma, bias = _statistics(g, 2, blocks)
    q, t = random(g, 2, 64), blocks * block_size + beyond
    given = [v.cuda() for v in (q, mean, std, gamma, bias)]
    at = torch.tensor([t, t], dtype=torch.int32, device="cuda")
    index, score = ba.route_blocks_rows(*given, torch.arange(2, dtype=torch.int32, device="cuda"), at, block_size, 2, top, False)
    same, same_score = ba.route_blocks(*given, torch.tensor(t, device="cuda"), block_size, 2, top, False)
    for b in range(2):
        want, value = plain.route(q[b], mean[b], std[b], gamma, bias, t, block_size, 2, top, False)
        assert index[b].tolist() == want == same[b].tolist()
        value = torch.tensor(value, dtype=torch.float64)
        within(score[b], value, 2.0 ** -24 * value.abs() + 1e-12)
    assert torch.equal(score, same_score)
    status_clear()


@pytest.mark.parametrize("strict", (False, True))
@pytest.mark.parametrize("window", (1, 40))
def test_route_chooses_by_the_scores_of_the_selectors(strict, window):
    import oracle

    batch, blocks, block_size, top = 3, 64, 16, 7
    g = torch.Generator().manual_seed(window)
    mean, std, gamma, bias = _statistics(g, batch, blocks)
    length = blocks * block_size
    q = random(g, batch * length, 64)
    index, score = (x.cpu() for x in ba.route_blocks_prefill(*[v.cuda() for v in (q, mean, std, gamma, bias)], length, block_size,
                                                             window, top, strict))
    for i in range(0, batch * length, 37):
        b, t = divmod(i, length)
        ours = oracle.block_scores(mean[b], std[b], q[i], gamma, bias, t, length, window, strict).double()
        # a head's score in 32 bits: 20 operations on the sum of its magnitudes, logarithms and exponentials to 2^-20
        size = (q[i].abs().view(4, 16) * mean[b].abs()).sum(-1) + torch.nn.functional.softplus(gamma) * (q[i].abs().view(4, 16) * std[b]).sum(-1)
        error = float((20 * 2.0 ** -24 * (size / 4 + bias.abs().amax())).max()) + 2.0 ** -19
        some = index[i] >= 0
        assert int(some.sum()) == min(top, int((ours > -math.inf).sum()))
        chosen = ours[index[i][some].long()]
        assert bool(((score[i][some].double() - chosen).abs() <= error).all())
        rest = ours.clone()
        rest[index[i][some].long()] = -math.inf
        assert bool((chosen >= rest.max() - 2 * error).all()) and bool((chosen[1:] <= chosen[:-1] + 2 * error).all())


@pytest.mark.parametrize("top", (1, 4))
def test_route_chooses_the_blocks_that_the_selector_looks_into(top):
    # every remote key scores the same and more than the window's one: the anchor is the first row of the first chosen block
    from relation_lm.kernels.relation_select import relation_select_packed

    batch, blocks, block_size, t = 8, 32, 16, 509
    g = torch.Generator().manual_seed(top)
    mean, std, gamma, bias = (v.cuda() for v in _statistics(g, batch, blocks))
    rq, query = random(g, batch, 64).cuda(), torch.ones(batch, 64, device="cuda")
    keys = torch.ones(batch, blocks * block_size, 64, device="cuda")
    keys[:, t] = -1.0
    partner = torch.zeros(batch, blocks * block_size, 128, device="cuda")
    position = torch.tensor(t, device="cuda")
    anchor = relation_select_packed(query, keys, rq, mean, std, gamma, bias, partner[:, 0].contiguous(), partner, keys, mean, std, gamma,
                                    bias, position, 1, top, 8, True)[0]
    index, _ = ba.route_blocks(rq, mean, std, gamma, bias, position, block_size, 1, top, True)
    assert torch.equal(anchor, index.amin(1) * block_size) and len(set(index.flatten().tolist())) > 4
    status_clear()


# ---------------------------------------------------------------------------- several rows a CTA


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form", ("rows", "prefill"))
@pytest.mark.parametrize("batch,length,heads,kv_heads,width,rotary,interleaved", [
    (3, 397, 8, 2, 64, 64, False), (1, 1184, 16, 4, 128, 64, True), (5, 1001, 2, 1, 64, 64, False), (2, 2999, 3, 3, 32, 16, True),
    (7, 2801, 1, 1, 8, 8, False), (3, 6667, 1, 1, 16, 0, False), (2, 3001, 1, 1, 7, 4, True), (1, 5003, 1, 1, 1024, 1024, False)])
def test_rotary_append_of_many_rows(dtype, form, batch, length, heads, kv_heads, width, rotary, interleaved):
    # as many rows as put several into a CTA, the last of which is short: bit for bit what a few rows at a time give
    g = torch.Generator().manual_seed(length)
    n = batch * length
    q, k, v = (random(g, n, h, width, dtype=dtype).cuda() for h in (heads, kv_heads, kv_heads))
    before = [random(g, batch, length + 3, kv_heads, width, dtype=dtype).cuda() for _ in range(2)]
    f, magnitude = ba.rotary_frequencies(rotary, scaling="by_parts", factor=2.0, trained_context=64)
    f = f.cuda()
    order = torch.randperm(n, generator=g) if form == "rows" else torch.arange(n)
    row_batch, row_position = (order // length).int(), (order % length).int()
    if form == "rows":
        row_position[order % 11 == 3] = -1               # rows of padding
    caches, few = [c.clone() for c in before], [c.clone() for c in before]
    rows = row_batch.cuda(), row_position.cuda()
    if form == "rows":
        out = ba.rotary_append_rows(q, k, v, *caches, f, *rows, interleaved, magnitude)
    else:
        out = ba.rotary_append_prefill(q, k, v, *caches, f, length, interleaved, magnitude)
    parts = [slice(i, min(i + 500, n)) for i in range(0, n, 500)]
    want = torch.cat([ba.rotary_append_rows(q[s], k[s], v[s], *few, f, *(r[s] for r in rows), interleaved, magnitude) for s in parts])
    assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(caches, few))
    for i in [0, 1, n - 1] + torch.randint(0, n, (20,), generator=g).tolist():
        b, t = int(row_batch[i]), int(row_position[i])
        if t < 0:
            assert not out[i].any()
            continue
        within(out[i], *plain.turned(q[i].cpu(), t, f.cpu(), interleaved, magnitude))
        within(caches[0][b, t], *plain.turned(k[i].cpu(), t, f.cpu(), interleaved, magnitude))
        assert torch.equal(caches[1][b, t], v[i])
    assert all(torch.equal(c[:, length:], o[:, length:]) for c, o in zip(caches, before))
    status_clear()


# ---------------------------------------------------------------------------- the three passes of whole sequences


def passes_of(q, k_cache, index, length, block_size, window):
    """The workspace of a whole-sequence call, in bytes: above zero where it takes the three passes, and of several launches
    where it is less than the partial results of all rows."""
    import ctypes

    from relation_lm.kernels import _abi

    size = ctypes.c_int64(-1)
    index = index if index.dim() == 3 else index[:, None].expand(-1, k_cache.size(2), -1)
    steps = (ctypes.c_int64 * 10)(*q.stride()[:2], *k_cache.stride()[:3], *k_cache.stride()[:3], *index.stride()[:2])
    assert _abi.LIB.rlm_block_attention_workspace(steps, q.size(0), k_cache.size(0), k_cache.size(1), length, q.size(1), k_cache.size(2),
                                                  q.size(2), index.size(2), block_size, window, _abi.code(q), ctypes.byref(size)) == 0
    return size.value


def _whole(seed, dtype, batch, length, heads, kv_heads, width, block_size, top):
    g = torch.Generator().manual_seed(seed)
    n = batch * length
    q = random(g, n, heads, width, dtype=dtype).cuda()
    caches = [random(g, batch, length, kv_heads, width, dtype=dtype).cuda() for _ in range(2)]
    t = torch.arange(length).repeat(batch)
    index = (torch.rand(n, kv_heads, top, generator=g) * (t[:, None, None] // block_size + 2)).int() - 1
    return q, *caches, index.cuda()


def _check_whole(x, length, block_size, window, scale, out, lse, every):
    q, k_cache, v_cache, index = (v.cpu() for v in x)
    at = [divmod(i, length) for i in range(q.size(0))]
    check_rows(range(0, q.size(0), every), at, q, k_cache, v_cache, index, out, lse, block_size, window, scale)


CASES = [(torch.bfloat16, 2, 601, 8, 2, 64, 64, 40, 3), (torch.float16, 1, 1100, 4, 2, 96, 32, 17, 5), (torch.float16, 2, 700, 8, 2, 128, 16, 0, 20)]


@pytest.mark.parametrize("case", CASES)
def test_three_passes_on_two_streams_at_once(case):
    dtype, batch, length, heads, kv_heads, width, block_size, window, top = case
    xs = [_whole(seed, dtype, batch, length, heads, kv_heads, width, block_size, top) for seed in range(2)]
    rest = (length, block_size, window, 0.125)
    assert all(passes_of(x[0], x[1], x[3], length, block_size, window) > 0 for x in xs)
    want = [ba.block_attention_prefill(*x, *rest) for x in xs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in xs], [[], []]
    for _ in range(12):
        for x, s, keep in zip(xs, streams, got):
            with torch.cuda.stream(s):
                keep.append(ba.block_attention_prefill(*x, *rest))
    torch.cuda.synchronize()
    for x, w, keep in zip(xs, want, got):
        _check_whole(x, *rest, *w, 97)
        assert all(torch.equal(a, b) for r in keep for a, b in zip(r, w))
    status_clear()


@pytest.mark.parametrize("case", CASES)
def test_three_passes_by_programmatic_launch(case):
    from relation_lm.kernels import _abi

    dtype, batch, length, heads, kv_heads, width, block_size, window, top = case
    x = _whole(3, dtype, batch, length, heads, kv_heads, width, block_size, top)
    assert passes_of(x[0], x[1], x[3], length, block_size, window) > 0
    f = ba.rotary_frequencies(width, device="cuda")[0]

    def layer():
        caches = [torch.zeros_like(c) for c in x[1:3]]
        q = ba.rotary_append_prefill(x[0], x[1].flatten(0, 1), x[2].flatten(0, 1), *caches, f, length)
        first = ba.block_attention_prefill(q, *caches, x[3], length, block_size, window, 0.125)
        return (q, *caches, *first, *ba.block_attention_prefill(first[0], *caches, x[3], length, block_size, window, 0.125))

    want, chained = layer(), _abi.programmatic_launch(layer)
    for _ in range(6):
        assert all(torch.equal(a, b) for a, b in zip(want, chained()))
    _check_whole((want[0], want[1], want[2], x[3]), length, block_size, window, 0.125, want[3], want[4], 97)
    status_clear()


@pytest.mark.parametrize("programmatic", (False, True))
def test_several_launches_over_one_workspace(programmatic):
    # more segments than fit the workspace: it is used again and again, also while the launch before it is still at its end
    from relation_lm.kernels import _abi

    batch, length, heads, kv_heads, width, block_size, window, top = 24, 1024, 16, 2, 128, 64, 33, 8
    x = _whole(5, torch.bfloat16, batch, length, heads, kv_heads, width, block_size, top)
    size = passes_of(x[0], x[1], x[3], length, block_size, window)
    assert 0 < size < batch * length * heads * top * width * 4 / 2
    call = _abi.programmatic_launch(ba.block_attention_prefill) if programmatic else ba.block_attention_prefill
    out, lse = call(*x, length, block_size, window, 0.0884)
    again, lse_again = call(*x, length, block_size, window, 0.0884)
    assert torch.equal(out, again) and torch.equal(lse, lse_again)
    for b in range(batch):                               # a sequence alone fits the workspace
        rows = slice(b * length, (b + 1) * length)
        alone, lse_alone = ba.block_attention_prefill(x[0][rows], x[1][b:b + 1], x[2][b:b + 1], x[3][rows], length, block_size, window, 0.0884)
        assert torch.equal(out[rows], alone) and torch.equal(lse[rows], lse_alone), b
    _check_whole(x, length, block_size, window, 0.0884, out, lse, 1777)
    status_clear()


@pytest.mark.parametrize("case", CASES)
def test_three_passes_in_captured_graphs(case):
    # two graphs of one memory pool, replayed in turn and with new inputs, and two graphs of their own at once
    dtype, batch, length, heads, kv_heads, width, block_size, window, top = case
    rest = (length, block_size, window, 0.125)
    xs = [_whole(seed, dtype, batch, length, heads, kv_heads, width, block_size, top) for seed in (7, 8)]
    fresh = [_whole(seed, dtype, batch, length, heads, kv_heads, width, block_size, top) for seed in (9, 10)]
    want, want_fresh = ([ba.block_attention_prefill(*x, *rest) for x in many] for many in (xs, fresh))
    assert passes_of(xs[0][0], xs[0][1], xs[0][3], length, block_size, window) > 0
    torch.cuda.synchronize()

    def capture(x, pool=None):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            out = ba.block_attention_prefill(*x, *rest)
        return graph, out

    first, out = capture(xs[0])
    second, out2 = capture(xs[1], first.pool())
    apart, out3 = capture(xs[1])
    for _ in range(3):
        for graph in (first, second):
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for r, w in zip((out, out2), want) for a, b in zip(r, w))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(6):
        for graph, s in zip((first, apart), streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r, w in zip((out, out3), want) for a, b in zip(r, w))
    for x, y in zip(xs, fresh):
        for a, b in zip(x, y):
            a.copy_(b)
    first.replay()
    second.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r, w in zip((out, out2), want_fresh) for a, b in zip(r, w))
    status_clear()


@pytest.mark.parametrize("dtype", HALF_TYPES)
def test_whole_sequence_layer_by_the_three_passes(dtype):
    """rotary_append -> router_cache_update -> route_blocks -> block_attention over whole sequences that are long enough for
    the passes, and the last positions of the same layer one by one."""
    from relation_lm.kernels.router_cache import router_cache_update

    batch, length, block, heads, kv_heads, width, window, top = 2, 800, 16, 4, 2, 64, 30, 3
    g = torch.Generator().manual_seed(12)
    n = batch * length
    q, k, v = (random(g, n, h, width, dtype=dtype).cuda() for h in (heads, kv_heads, kv_heads))
    rq, rk = random(g, n, 64, dtype=dtype).cuda(), random(g, batch, length, 64, dtype=dtype).cuda()
    conv, gamma, bias = random(g, 64, 3, scale=0.1).cuda(), random(g, 4).cuda(), random(g, 4, 8).cuda()
    f, magnitude = ba.rotary_frequencies(width, scaling="by_parts", factor=2.0, trained_context=400, device="cuda")
    caches = [torch.zeros(batch, length, kv_heads, width, device="cuda", dtype=dtype) for _ in range(2)]
    turned = ba.rotary_append_prefill(q, k, v, *caches, f, length, True, magnitude)
    router = ([torch.zeros(batch, length, 64, device="cuda", dtype=dtype) for _ in range(4)]
              + [torch.zeros(batch, length // block, 4, 16, device="cuda", dtype=dtype) for _ in range(4)])
    for t in range(length):
        router_cache_update(rk[:, t].contiguous(), rk[:, t].contiguous(), *router, conv, conv, torch.tensor(t, device="cuda"), block)
    index, score = ba.route_blocks_prefill(rq, router[4], router[5], gamma, bias, length, block, window, top, True)
    assert passes_of(turned, caches[0], index, length, block, window) > 0
    out, lse = ba.block_attention_prefill(turned, *caches, index, length, block, window, 0.125)
    for t in (length - 1, length - 17, 401, 30, 0):
        rows = torch.arange(batch, device="cuda") * length + t
        at = torch.tensor(t, device="cuda")
        step = ba.rotary_append(q[rows], k[rows], v[rows], *[torch.zeros_like(c) for c in caches], f, at, True, magnitude)
        assert torch.equal(step, turned[rows])
        one, one_score = ba.route_blocks(rq[rows], router[4], router[5], gamma, bias, at, block, window, top, True)
        assert torch.equal(one, index[rows]) and torch.equal(one_score, score[rows])
        step_out, step_lse = ba.block_attention(step, *caches, one, at, block, window, 0.125)
        for b in range(batch):
            want, want_lse, bound, lse_bound = plain.attend(step[b].cpu(), caches[0][b].cpu(), caches[1][b].cpu(), one[b].cpu().expand(2, -1), t,
                                                            block, window, 0.125)
            for y, z in ((step_out[b], step_lse[b]), (out[rows[b]], lse[rows[b]])):
                within(y, want, bound, t)
                within(z, want_lse, lse_bound, t)
    status_clear()


@pytest.mark.parametrize("gamma,query,spread", [(1e22, 1e-23, 750.0), (1e25, 1e-12, 7.5e-11), (3e9, 1e-23, 2.0e16), (750.0, 1.0, 1.0)])
@pytest.mark.parametrize("form", ("decode", "rows", "prefill"))
def test_the_choice_is_that_of_64_bits_at_any_magnitude(form, gamma, query, spread):
    # tiny queries under a steep factor: scores of hundreds whose magnitudes' squares vanish in 32 bits; blocks differ by the last
    # bits of their spreads, less than what a score in 32 bits is off by
    blocks, top = (1000, 9) if form != "prefill" else (120, 9)
    g = torch.Generator().manual_seed(3)
    step = torch.finfo(torch.float32).eps * 2.0 ** math.floor(math.log2(spread))
    mean = torch.zeros(1, blocks, 4, 16)
    std = (spread + torch.randint(0, 4, (1, blocks, 4, 16), generator=g).double() * step).float()
    n = {"decode": 1, "rows": 600, "prefill": 9000}[form]
    q = (query * (0.5 + 0.5 * torch.rand(n, 64, generator=g).double())).float()
    at = plain.places(form, 1, 0, 0, n) if form == "prefill" else [(0, 4 * blocks - 1 - i) for i in range(n)]
    size = 64 if form == "prefill" else 4
    call = {"decode": ba.route_blocks, "rows": ba.route_blocks_rows, "prefill": ba.route_blocks_prefill}[form]
    scales = torch.full((4,), gamma), torch.zeros(4, 1)
    index, score = call(q.cuda(), mean.cuda(), std.cuda(), *[v.cuda() for v in scales], *plain.where(form, at, n), size, 0, top, False)
    soft = float(scales[0][0].double())                  # softplus of factors this large, to less than 1e-300
    for i in sorted({0, n // 3, n // 2, n - 2, n - 1}):
        able = min((at[i][1] + 1) // size, blocks)
        heads = soft * (q[i].double().view(4, 16) * std[0, :able].double()).sum(-1) / 4
        value = torch.logsumexp(heads, 1)
        want = sorted(range(able), key=lambda b: (-float(value[b]), b))[:top]
        assert index[i].tolist() == want + [-1] * (top - len(want)), i
        within(score[i][:len(want)], value[want], 2.0 ** -24 * value[want].abs() + 1e-12)
    status_clear()
