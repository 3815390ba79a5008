"""The serving operators on the GPU against their definitions in 64 bits: appending to a paged cache, attention over it, rules on
logits, and the three in one step."""
import ctypes
import math

import numpy as np
import pytest
import torch
from serving_utils import (BAD_INDEX, Cache, append, append_args, attention, attention_args, attention_exact, attention_tolerance, i32, lib,
                           power_of_two, ptr, rope_tables, rotated, rules, rules_args, starts, status, workspace)

pytestmark = pytest.mark.gpu
KINDS = ["bf16", "e4m3"]


def qkv_rows(n, heads, kv, hd, seed, pad=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, (heads + 2 * kv) * hd + pad, generator=g)
    x *= torch.exp(0.7 * torch.randn(1, x.shape[1], generator=g))
    return x.to(torch.bfloat16).cuda()


# ---- append -------------------------------------------------------------------------------------------------------------------
def check_append(kind, heads, kv, hd, page, new, pos, pad=0, extra=0, before=0, behind=0, rotate=True, seed=1):
    start = starts(new, before)
    n = start[-1] + behind
    cache = Cache([p + a for p, a in zip(pos, new)], kv, hd, page, kind, seed=seed, extra=extra)
    qkv = qkv_rows(n, heads, kv, hd, seed, pad)
    q = torch.full((n, heads * hd + pad), 7.0, dtype=torch.bfloat16, device="cuda")
    cos, sin = rope_tables(max(p + a for p, a in zip(pos, new)) + 1, hd) if rotate else (None, None)
    old = {"k": cache.k.clone(), "v": cache.v.clone(), "ks": None if cache.ks is None else cache.ks.clone(),
           "vs": None if cache.vs is None else cache.vs.clone()}
    append(cache, heads, qkv, q, i32(start), i32(pos), cos, sin)
    torch.cuda.synchronize()
    assert status() == 0

    x = qkv[:, :(heads + 2 * kv) * hd].float().cpu().view(n, -1, hd)
    at = torch.zeros(n, dtype=torch.long)
    owner = torch.full((n,), -1)
    for b in range(len(new)):
        at[start[b]:start[b + 1]] = torch.arange(pos[b], pos[b] + new[b])
        owner[start[b]:start[b + 1]] = b
    if rotate:
        f32, f64 = rotated(x[:, :heads + kv], cos.cpu()[at], sin.cpu()[at])
    else:
        f32, f64 = x[:, :heads + kv], x[:, :heads + kv].double()
    mag = x[:, :heads + kv].abs().double().view(n, heads + kv, hd // 2, 2).sum(-1).repeat_interleave(2, -1)
    mine = owner >= 0
    # queries: one rounding to bf16 of a sum of two fp32 products
    got = q[:, :heads * hd].double().cpu().view(n, heads, hd)
    assert ((got - f64[:, :heads]).abs() <= 2.0 ** -8 * f64[:, :heads].abs() + 2.0 ** -22 * mag[:, :heads])[mine].all()
    # what belongs to nobody stays
    assert (q[~mine.cuda()] == 7).all() and (q[:, heads * hd:] == 7).all()
    for name, r32, r64, m in (("k", f32[:, heads:], f64[:, heads:], mag[:, heads:]), ("v", x[:, heads + kv:], x[:, heads + kv:].double(), 0)):
        was, now = old[name], getattr(cache, name)
        assert torch.equal(was[:, kv * page * hd:].view(torch.uint8), now[:, kv * page * hd:].view(torch.uint8))
        want = cache.blocks(was).cpu().float().double()
        tol = torch.zeros_like(want)
        same = torch.ones(cache.pages, kv, page, dtype=torch.bool)  # rows that keep their bytes
        scales = None
        if kind == "e4m3":
            scales = old[name + "s"].cpu().double()
        for b in range(len(new)):
            for p0 in range(pos[b] // page * page, pos[b] + new[b], page) if new[b] else []:
                pg = cache.table_host[b][p0 // page]
                lo, hi = max(pos[b], p0), min(pos[b] + new[b], p0 + page)
                rows = slice(start[b] + lo - pos[b], start[b] + hi - pos[b])
                part64, part32 = r64[rows].transpose(0, 1), r32[rows]
                span = slice(lo - p0, hi - p0)
                same[pg, :, span] = False
                slack = 2.0 ** -22 * m[rows].transpose(0, 1) if isinstance(m, torch.Tensor) else 0.0
                if kind == "bf16":
                    want[pg, :, span] = part64
                    tol[pg, :, span] = 2.0 ** -8 * part64.abs() + slack
                    continue
                need = torch.from_numpy(power_of_two(part32.abs().amax((0, 2)).numpy()).astype(np.float64))
                before_scale = scales[pg].clone() if lo > p0 else torch.zeros(kv, dtype=torch.float64)
                scales[pg] = torch.maximum(before_scale, need)
                s = scales[pg][:, None, None]
                if lo > p0:
                    ratio = (before_scale / scales[pg])[:, None, None]
                    held = want[pg, :, :lo - p0] * ratio
                    # powers of two: what is normal keeps its bits, what is not is off by half a subnormal step
                    tol[pg, :, :lo - p0] = torch.where((held.abs() >= 2.0 ** -6) | (ratio == 1), 0.0, 2.0 ** -10).expand_as(held)
                    want[pg, :, :lo - p0] = held
                    same[pg, :, :lo - p0] = (ratio == 1)[:, :, 0].expand(-1, lo - p0)
                want[pg, :, span] = part64 / s
                tol[pg, :, span] = 2.0 ** -4 * (part64 / s).abs() + 2.0 ** -10 + slack / s
        if kind == "e4m3":
            assert torch.equal(getattr(cache, name + "s").cpu().double(), scales)
        got = cache.blocks(now).cpu().float().double()
        assert ((got - want).abs() <= tol).all(), float(((got - want).abs() - tol).max())
        assert torch.equal(cache.blocks(now).cpu().view(torch.uint8).view(cache.pages, kv, page, -1)[same],
                           cache.blocks(was).cpu().view(torch.uint8).view(cache.pages, kv, page, -1)[same])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,hd,page", [(12, 12, 64, 16), (12, 4, 64, 64), (6, 6, 48, 48), (4, 1, 128, 128), (8, 1, 32, 32), (12, 4, 96, 16)])
@pytest.mark.parametrize("new,pos", [
    ([1], [0]),
    ([1, 1, 1], [15, 16, 17]),
    ([1] * 9, [0, 1, 63, 64, 65, 100, 127, 128, 300]),
    ([5, 0, 130, 1], [3, 40, 0, 63]),
    ([200, 33], [1, 95]),
])
def test_append_matches_its_definition(kind, heads, kv, hd, page, new, pos):
    check_append(kind, heads, kv, hd, page, new, pos)


@pytest.mark.parametrize("kind", KINDS)
def test_append_leaves_what_is_not_its_own(kind):
    # padded rows and pages, rows before the first and behind the last sequence
    check_append(kind, 8, 2, 64, 32, [3, 40, 1], [30, 5, 64], pad=24, extra=48, before=2, behind=5)
    check_append(kind, 8, 2, 64, 32, [3, 40, 1], [30, 5, 64], rotate=False)


@pytest.mark.parametrize("kind", KINDS)
def test_append_in_place_and_without_queries(kind):
    heads, kv, hd, new, pos = 4, 2, 64, [7, 1], [3, 50]
    cos, sin = rope_tables(64, hd)
    qkv = qkv_rows(8, heads, kv, hd, 3)
    caches = [Cache([10, 51], kv, hd, 16, kind, seed=2) for _ in range(3)]
    q = torch.empty(8, heads * hd, dtype=torch.bfloat16, device="cuda")
    append(caches[0], heads, qkv, q, i32(starts(new)), i32(pos), cos, sin)
    keep = qkv.clone()
    append(caches[1], heads, qkv, None, i32(starts(new)), i32(pos), cos, sin)
    assert torch.equal(keep, qkv)
    append(caches[2], heads, qkv, qkv, i32(starts(new)), i32(pos), cos, sin)
    assert torch.equal(qkv[:, :heads * hd], q) and torch.equal(qkv[:, heads * hd:], keep[:, heads * hd:])
    for c in caches[1:]:
        assert torch.equal(c.k.view(torch.uint8), caches[0].k.view(torch.uint8))
        assert torch.equal(c.v.view(torch.uint8), caches[0].v.view(torch.uint8))


def test_append_token_by_token_gives_what_one_call_gives():
    """Powers of two: normal values do not depend on how a page came about, others by half a step of the final scale for each growth."""
    heads, kv, hd, page, n = 2, 2, 64, 32, 70
    cos, sin = rope_tables(n, hd)
    qkv = qkv_rows(n, heads, kv, hd, 5)
    qkv[:, heads * hd:] *= torch.exp2(torch.arange(n, device="cuda") / 8)[:, None].to(torch.bfloat16)  # scales keep growing
    one, many = (Cache([n], kv, hd, page, "e4m3", seed=4, fill=False) for _ in range(2))
    append(one, heads, qkv, None, i32([0, n]), i32([0]), cos, sin)
    for t in range(n):
        append(many, heads, qkv[t:t + 1], None, i32([0, 1]), i32([t]), cos, sin)
    for name in ("k", "v"):
        assert torch.equal(getattr(one, name + "s")[one.table[0, :3].long()], getattr(many, name + "s")[one.table[0, :3].long()])
        a, b = one.rows(name, 0, n), many.rows(name, 0, n)
        s = getattr(one, name + "s").cpu().double()[torch.tensor(one.table_host[0])[torch.arange(n) // page]][..., None]
        # every growth at least halves what a rounding before it left: in all less than twice half a subnormal step, a side
        assert ((a - b).abs() <= torch.where(a.abs() >= 2.0 ** -5 * s, 0.0, 2.0 ** -8 * s)).all()


def test_append_infinite_nan_and_zero_values():
    heads, kv, hd = 1, 1, 32
    cache = Cache([16], kv, hd, 16, "e4m3", fill=False)
    qkv = torch.zeros(16, 3 * hd, dtype=torch.bfloat16, device="cuda")
    append(cache, heads, qkv, None, i32([0, 16]), i32([0]), None, None)
    pg = cache.table_host[0][0]
    assert float(cache.ks[pg, 0]) == 2.0 ** -126 and float(cache.k.float().abs().max()) == 0
    qkv[0, hd], qkv[1, hd], qkv[2, hd], qkv[3, hd] = math.inf, -math.inf, math.nan, 3.0
    append(cache, heads, qkv, None, i32([0, 16]), i32([0]), None, None)
    got = cache.rows("k", 0, 16)[:, 0, 0]
    assert float(cache.ks[pg, 0]) == 2.0 ** -7  # 3 / 448 = 0.0067
    assert got[0] == 448 * 2.0 ** -7 and got[1] == -448 * 2.0 ** -7 and math.isnan(got[2]) and got[3] == 3.0
    qkv[:, hd] = 448.0  # the largest value that the scale 1 takes
    append(cache, heads, qkv, None, i32([0, 16]), i32([0]), None, None)
    assert float(cache.ks[pg, 0]) == 1.0 and (cache.rows("k", 0, 16)[:, 0, 0] == 448).all()


@pytest.mark.parametrize("kind", KINDS)
def test_append_out_of_range_is_not_written(kind):
    heads, kv, hd, page = 2, 2, 64, 16
    cos, sin = rope_tables(40, hd)
    qkv = qkv_rows(4, heads, kv, hd, 6)

    def attempt(start, pos, table=None, n_seq=None):
        cache = Cache([32, 32], kv, hd, page, kind, seed=3)
        if table is not None:
            cache.table.copy_(i32(table))
        k, v = cache.k.clone(), cache.v.clone()
        q = torch.zeros(4, heads * hd, dtype=torch.bfloat16, device="cuda")
        append(cache, heads, qkv, q, i32(start), i32(pos), cos, sin)
        code = status()
        return code, torch.equal(k.view(torch.uint8), cache.k.view(torch.uint8)) and torch.equal(v.view(torch.uint8), cache.v.view(torch.uint8))

    assert attempt([0, 2, 4], [0, 16])[0] == 0
    assert attempt([0, 4], [48 - 3]) == (BAD_INDEX, True)               # one token more than the table has room for
    assert attempt([0, 4], [-1]) == (BAD_INDEX, True)
    assert attempt([-1, 3], [0]) == (BAD_INDEX, True)
    assert attempt([0, 5], [0]) == (BAD_INDEX, True)                    # rows that are not there
    assert attempt([0, 4], [0], [[7, 0, 0], [0, 0, 0]]) == (BAD_INDEX, True)   # pages are 0 .. 6
    assert attempt([0, 4], [0], [[-1, 0, 0], [0, 0, 0]]) == (BAD_INDEX, True)
    assert attempt([0, 4], [2 ** 31 - 2]) == (BAD_INDEX, True)
    assert attempt([0, 0, 0], [0, 16]) == (0, True)                     # no tokens at all


# ---- attention ----------------------------------------------------------------------------------------------------------------
def check_attention(kind, heads, kv, hd, page, new, pos, window=0, scale=0.0, pad=0, extra=0, before=0, behind=0, seed=1, loud=1.0, cache=None,
                    hidden_nan=True):
    start = starts(new, before)
    n = start[-1] + behind
    g = torch.Generator().manual_seed(seed + 100)
    if cache is None:
        cache = Cache([p + a for p, a in zip(pos, new)], kv, hd, page, kind, seed=seed, extra=extra)
    if hidden_nan:  # what lies behind a sequence's end in its last page
        for name in ("k", "v"):
            blocks = cache.blocks(getattr(cache, name)).clone().view(torch.uint8).view(cache.pages, kv, page, -1)
            for b, (p, a) in enumerate(zip(pos, new)):
                if (p + a) % page:
                    blocks[cache.table_host[b][(p + a) // page], :, (p + a) % page:] = 0xff
            raw = getattr(cache, name).view(torch.uint8)
            raw[:, :blocks[0].numel()] = blocks.reshape(cache.pages, -1)
    q = (1.5 * loud * torch.randn(n, heads * hd + pad, generator=g)).to(torch.bfloat16).cuda()
    out = torch.full((n, heads * hd + pad), 7.0, dtype=torch.bfloat16, device="cuda")
    attention(cache, heads, q, out, i32(start), i32(pos), max(max(new), 1), window=window, scale=scale)
    torch.cuda.synchronize()
    assert status() == 0
    mine = torch.zeros(n, dtype=torch.bool)
    mine[start[0]:start[-1]] = True
    assert (out[~mine.cuda()] == 7).all() and (out[:, heads * hd:] == 7).all()
    factor = scale or hd ** -0.5
    for b, (p, a) in enumerate(zip(pos, new)):
        if not a:
            continue
        mq = q[start[b]:start[b + 1], :heads * hd].double().cpu().view(a, heads, hd)
        k, v = cache.rows("k", b, p + a), cache.rows("v", b, p + a)
        ref, mass, big = attention_exact(mq, k, v, p, factor, window)
        got = out[start[b]:start[b + 1], :heads * hd].double().cpu().view(a, heads, hd)
        tol = attention_tolerance(ref, mass, big, kind, hd, p + a, mq, factor, float(k.abs().max()))
        assert ((got - ref).abs() <= tol).all(), (b, float(((got - ref).abs() - tol).max()), float((got - ref).norm() / ref.norm()))
    return cache, q, out


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,hd,page", [(12, 12, 64, 16), (12, 4, 64, 64), (6, 6, 48, 48), (16, 1, 128, 128), (8, 1, 32, 32), (12, 4, 96, 16),
                                              (40, 2, 128, 16)])
@pytest.mark.parametrize("new,pos", [
    ([1], [0]),
    ([1, 1, 1, 1], [14, 15, 16, 400]),
    ([1, 0, 1], [2500, 3, 63]),
    ([2, 5, 3], [63, 0, 700]),
    ([37, 1, 90], [100, 12, 0]),
])
def test_attention_matches_its_definition(kind, heads, kv, hd, page, new, pos):
    check_attention(kind, heads, kv, hd, page, new, pos)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window", [1, 16, 100, 1000])
@pytest.mark.parametrize("new,pos", [([1, 1], [0, 1500]), ([3, 20], [170, 3]), ([70], [900])])
def test_attention_window(kind, window, new, pos):
    check_attention(kind, 8, 2, 64, 16, new, pos, window=window)


@pytest.mark.parametrize("kind", KINDS)
def test_attention_strides_scale_and_rows_of_nobody(kind):
    check_attention(kind, 8, 2, 64, 32, [3, 40, 1], [30, 5, 640], pad=24, extra=48, before=2, behind=5, scale=0.3)
    check_attention(kind, 8, 2, 64, 32, [1, 1], [3000, 1], pad=8, behind=1)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("loud", [1e-3, 30.0])
def test_attention_flat_and_sharp_softmax(kind, loud):
    check_attention(kind, 4, 2, 64, 16, [1, 6, 20], [1000, 900, 64], loud=loud)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [1, 8, 40])
def test_attention_of_many_shared_parts(kind, new):
    # one long sequence over all CTAs, beside short ones
    check_attention(kind, 4, 1, 64, 128, [new, 1, new, 1], [30001, 5, 4097, 300])


def test_attention_scales_of_any_size_and_mixed():
    cache = Cache([2000], 2, 64, 16, "e4m3", seed=9)
    g = torch.Generator().manual_seed(5)
    # values of very different pages, and scales that are no powers of two
    cache.vs.copy_((torch.rand(cache.vs.shape, generator=g) * 10.0 ** torch.randint(-6, 4, cache.vs.shape, generator=g)).cuda())
    cache.ks.copy_((cache.ks.cpu() * (0.5 + torch.rand(cache.ks.shape, generator=g))).cuda())
    check_attention("e4m3", 4, 2, 64, 16, [1], [1999], cache=cache)


@pytest.mark.parametrize("new", [1, 40, 100])
def test_attention_pages_of_zeros_and_of_the_smallest_values(new):
    # the scale of a page of zeros is 2^-126, the smallest that appending gives
    heads, kv, hd, n = 2, 1, 64, 200 + new
    cache = Cache([n], kv, hd, 16, "e4m3", fill=False)
    qkv = torch.zeros(n, (heads + 2) * hd, dtype=torch.bfloat16, device="cuda")
    qkv[:, :heads * hd] = 1.0
    start, pos = i32([0, n]), i32([0])
    append(cache, heads, qkv, None, start, pos, None, None)
    q = qkv[200:, :heads * hd].contiguous()
    out = torch.full_like(q, 7.0)
    attention(cache, heads, q, out, i32([0, new]), i32([200]), new)
    assert (out == 0).all()
    tiny = 2.0 ** -125  # 1 or 2 in units of the scale: a bf16 and an e4m3 number
    qkv[:, (heads + 1) * hd:] = tiny
    append(cache, heads, qkv, None, start, pos, None, None)
    attention(cache, heads, q, out, i32([0, new]), i32([200]), new)
    assert status() == 0
    assert ((out.double() / tiny - 1).abs() <= 2.0 ** -7).all()  # equal probabilities in 16 bits and their sums, rounded to bf16


@pytest.mark.parametrize("kind", KINDS)
def test_sequences_may_share_full_pages(kind):
    heads, kv, hd, page = 4, 2, 64, 16
    cache = Cache([100, 100, 100], kv, hd, page, kind, seed=6)
    for b in (1, 2):  # three sequences with the same first 64 tokens
        for i in range(4):
            cache.table_host[b][i] = cache.table_host[0][i]
    cache.table = i32(cache.table_host)
    check_attention(kind, heads, kv, hd, page, [1, 3, 20], [70, 64, 66], cache=cache)


@pytest.mark.parametrize("kind", KINDS)
def test_two_streams_at_once(kind):
    heads, kv, hd = 8, 2, 64
    caches = [Cache([9000, 3000], kv, hd, 64, kind, seed=i) for i in range(2)]
    q = [torch.randn(2, heads * hd, generator=torch.Generator().manual_seed(i)).to(torch.bfloat16).cuda() for i in range(2)]
    start, pos = i32([0, 1, 2]), i32([8999, 2999])
    want = [torch.empty_like(x) for x in q]
    for i in range(2):
        attention(caches[i], heads, q[i], want[i], start, pos, 1)
    works, streams = [workspace(heads, kv, hd) for _ in range(2)], [torch.cuda.Stream() for _ in range(2)]
    got = [[torch.empty_like(x) for _ in range(20)] for x in q]
    torch.cuda.synchronize()
    for k in range(20):
        for i in range(2):
            attention(caches[i], heads, q[i], got[i][k], start, pos, 1, work=works[i], stream=streams[i].cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [1, 4, 40])
def test_attention_does_not_see_infinite_values_ahead(kind, new):
    """Keys and values that a query does not see may be anything: also those of later tokens of the same call, and behind a window."""
    heads, kv, hd, page, pos, window = 4, 2, 64, 16, 100, 60
    clean, q, want = check_attention(kind, heads, kv, hd, page, [new], [pos], window=window, hidden_nan=False)
    # spoil everything that the first `half` queries do not see
    half = max(1, new // 2)
    for name in ("k", "v"):
        blocks = clean.blocks(getattr(clean, name)).clone()
        for p in [*range(0, pos - window + 1), *range(pos + half, pos + new)]:
            pg = clean.table_host[0][p // page]
            if kind == "bf16":
                blocks[pg, :, p % page, ::3] = math.inf
                blocks[pg, :, p % page, 1::3] = math.nan
            else:
                blocks.view(torch.uint8)[pg, :, p % page, ::2] = 0x7f
        getattr(clean, name)[:, :blocks[0].numel()] = blocks.reshape(clean.pages, -1)
    out = torch.empty_like(want)
    attention(clean, heads, q, out, i32([0, new]), i32([pos]), new, window=window)
    a, b = out[:half].double().cpu(), want[:half].double().cpu()
    # the same sums in another order at most: both are within the tolerance of the same exact result
    k, v = clean.rows("k", 0, pos + half), clean.rows("v", 0, pos + half)
    k[:pos - window + 1], v[:pos - window + 1] = 0, 0
    ref, mass, big = attention_exact(q[:half].double().cpu().view(half, heads, hd), k, v, pos, hd ** -0.5, window)
    tol = attention_tolerance(ref, mass, big, kind, hd, pos + half, q.double().cpu(), hd ** -0.5, float(k.abs().max())).reshape(half, -1)
    assert torch.isfinite(a).all() and ((a - ref.reshape(half, -1)).abs() <= tol).all() and ((b - ref.reshape(half, -1)).abs() <= tol).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [1, 40])
def test_attention_visible_nan_reaches_its_row_only(kind, new):
    heads, kv, hd, page, pos = 2, 1, 64, 16, 50
    cache = Cache([pos + new], kv, hd, page, kind, seed=3)
    p = pos + new - 1  # the last token's own value, which only the last query sees
    raw = cache.v.view(torch.uint8)
    es = 2 if kind == "bf16" else 1
    at = (p % page) * hd * es
    raw[cache.table_host[0][p // page], at:at + es] = 0x7f
    if kind == "bf16":
        raw[cache.table_host[0][p // page], at:at + 2] = torch.tensor([0xc0, 0x7f], dtype=torch.uint8, device="cuda")
    q = torch.randn(new, heads * hd).to(torch.bfloat16).cuda()
    out = torch.empty_like(q)
    attention(cache, heads, q, out, i32([0, new]), i32([pos]), new)
    nan = torch.isnan(out.float().view(new, heads, hd)).cpu()
    assert nan[-1, :, 0].all() and nan.sum() == heads


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,hd,page", [(8, 1, 32, 16), (6, 6, 48, 48), (12, 4, 64, 64), (12, 4, 96, 16), (16, 2, 128, 32)])
@pytest.mark.parametrize("window", [0, 130])
def test_attention_of_prompts(kind, heads, kv, hd, page, window):
    # tiles of rows that end inside a sequence, keys from none before to many, prompts beside single tokens
    check_attention(kind, heads, kv, hd, page, [150, 33, 1, 0, 260], [700, 0, 64, 9, 5], window=window)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,hd", [(8, 1, 32), (4, 2, 96), (8, 1, 128)])
def test_attention_of_prompts_in_many_shared_parts(kind, heads, kv, hd):
    check_attention(kind, heads, kv, hd, 64, [70, 9], [20001, 300])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", [32, 48, 64, 96, 128])
@pytest.mark.parametrize("pos,at", [(0, 40), (0, 99), (300, 350)])
def test_attention_of_prompts_nan_reaches_later_rows_only(kind, hd, pos, at):
    """A value that is NaN, of a token of the prompt: rows before it are what they are without it, its own and later ones have a NaN in its column."""
    heads, kv, page, new = 6, 2, 64, 100
    cache, q, want = check_attention(kind, heads, kv, hd, page, [new], [pos], hidden_nan=False)
    es, column = (2, hd - 1) if kind == "bf16" else (1, hd - 1)
    first = (at % page) * hd * es + column * es  # of KV head 0
    cache.v.view(torch.uint8)[cache.table_host[0][at // page], first:first + es] = torch.tensor([0xc0, 0x7f][-es:], dtype=torch.uint8, device="cuda")
    out = torch.full_like(want, 7.0)
    attention(cache, heads, q, out, i32([0, new]), i32([pos]), new)
    assert status() == 0
    nan = torch.isnan(out.float()).view(new, heads, hd).cpu()
    assert nan[at - pos:, :heads // kv, column].all() and int(nan.sum()) == (new - (at - pos)) * (heads // kv)
    # the tile's products are summed one by one instead: rounding of probabilities is the same, the order of sums is not
    k, v = cache.rows("k", 0, pos + new), cache.rows("v", 0, pos + new)
    v[at] = 0
    mq = q.double().cpu().view(new, heads, hd)
    ref, mass, big = attention_exact(mq, k, v, pos, hd ** -0.5, 0)
    tol = attention_tolerance(ref, mass, big, kind, hd, pos + new, mq, hd ** -0.5, float(k.abs().max()))
    before = slice(0, at - pos)
    assert ((out.double().cpu().view(new, heads, hd) - ref).abs() <= tol)[before].all()


@pytest.mark.parametrize("kind", KINDS)
def test_a_captured_prompt_replayed_at_other_places(kind):
    heads, kv, hd, new = 8, 2, 64, 90
    cache = Cache([700], kv, hd, 64, kind, seed=6)
    q = torch.randn(new, heads * hd, generator=torch.Generator().manual_seed(6)).to(torch.bfloat16).cuda()
    want, out, work = torch.empty_like(q), torch.empty_like(q), workspace(heads, kv, hd)
    start, pos, stream = i32([0, new]), i32([0]), torch.cuda.Stream()
    attention(cache, heads, q, want, start, pos, new, work=work)  # and everything that a first call does
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        attention(cache, heads, q, out, start, pos, new, work=work, stream=stream.cuda_stream)
    for at in (0, 37, 610):
        pos.fill_(at)
        attention(cache, heads, q, want, start, pos, new, work=work)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert status() == 0 and torch.equal(out, want)


def test_prompts_of_two_head_sizes_on_two_streams():
    sizes = [(4, 1, 64, "bf16"), (4, 1, 128, "e4m3")]
    caches = [Cache([2100, 700], kv, hd, 64, kind, seed=i) for i, (_, kv, hd, kind) in enumerate(sizes)]
    q = [torch.randn(200, h * hd, generator=torch.Generator().manual_seed(i)).to(torch.bfloat16).cuda() for i, (h, _, hd, _) in enumerate(sizes)]
    start, pos = i32([0, 100, 200]), i32([2000, 600])
    want = [torch.empty_like(x) for x in q]
    for i, (h, _, _, _) in enumerate(sizes):
        attention(caches[i], h, q[i], want[i], start, pos, 100)
    works, streams = [workspace(h, kv, hd) for h, kv, hd, _ in sizes], [torch.cuda.Stream() for _ in sizes]
    got = [[torch.empty_like(x) for _ in range(20)] for x in q]
    torch.cuda.synchronize()
    for k in range(20):
        for i, (h, _, _, _) in enumerate(sizes):
            attention(caches[i], h, q[i], got[i][k], start, pos, 100, work=works[i], stream=streams[i].cuda_stream)
    torch.cuda.synchronize()
    assert status() == 0 and all(torch.equal(g, want[i]) for i in range(2) for g in got[i])


def test_attention_offsets_beyond_32_bits():
    # pages 2^28 bytes apart: the last ones begin behind 2^32
    kv, hd, page, pages, stride = 1, 64, 16, 20, 1 << 28
    cache = Cache([64], kv, hd, page, "e4m3", seed=3)
    k = torch.zeros(pages * stride, dtype=torch.uint8, device="cuda")
    ids = [19, 3, 18, 17]
    small = Cache([64], kv, hd, page, "e4m3", seed=3)
    for i, pg in enumerate(ids):
        k[pg * stride:pg * stride + page * hd] = small.blocks(small.k).view(torch.uint8)[small.table_host[0][i]].reshape(-1)
    v = k.clone()
    cache.k, cache.v = k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn)
    cache.stride, cache.pages = stride, pages
    cache.table = i32([ids])
    cache.pitch = 4
    cache.ks, cache.vs = (torch.full((pages, kv), 2.0 ** -7, device="cuda") for _ in range(2))
    small.v = small.k.clone()
    small.ks, small.vs = (torch.full_like(small.ks, 2.0 ** -7) for _ in range(2))
    q = torch.randn(1, 2 * hd).to(torch.bfloat16).cuda()
    out, want = torch.empty_like(q), torch.empty_like(q)
    attention(cache, 2, q, out, i32([0, 1]), i32([63]), 1)
    attention(small, 2, q, want, i32([0, 1]), i32([63]), 1)
    assert torch.equal(out, want)
    qkv = qkv_rows(20, 2, kv, hd, 6)
    append(cache, 2, qkv, None, i32([0, 20]), i32([40]), None, None)
    append(small, 2, qkv, None, i32([0, 20]), i32([40]), None, None)
    assert status() == 0
    for big, little in ((k, small.k), (v, small.v)):
        for i, pg in enumerate(ids):
            assert torch.equal(big[pg * stride:pg * stride + page * hd], small.blocks(little).view(torch.uint8)[small.table_host[0][i]].reshape(-1))


def test_attention_out_of_range_is_reported():
    heads, kv, hd, page = 2, 2, 64, 16
    cache = Cache([32, 32], kv, hd, page, "bf16", seed=3)
    q = torch.randn(4, heads * hd).to(torch.bfloat16).cuda()

    def attempt(start, pos, max_new=4, table=None):
        keep = cache.table.clone()
        if table:
            cache.table.copy_(i32(table))
        out = torch.full_like(q, 7.0)
        attention(cache, heads, q, out, i32(start), i32(pos), max_new)
        cache.table.copy_(keep)
        return status(), bool((out == 7).all())

    assert attempt([0, 1, 2], [5, 7])[0] == 0
    assert attempt([0, 4], [45]) == (BAD_INDEX, True)
    assert attempt([0, 4], [-3]) == (BAD_INDEX, True)
    assert attempt([0, 5], [0]) == (BAD_INDEX, True)
    assert attempt([0, 4], [0], max_new=3) == (BAD_INDEX, True)
    assert attempt([3, 1], [0]) == (BAD_INDEX, True)
    assert attempt([0, 0], [0]) == (0, True)
    assert attempt([0, 1, 2], [5, 7], table=[[7, 0, 0], [1, 2, 3]])[0] == BAD_INDEX
    assert attempt([0, 1, 2], [20, 7], table=[[0, -1, 0], [1, 2, 3]])[0] == BAD_INDEX


@pytest.mark.parametrize("kind", KINDS)
def test_attention_is_the_same_from_call_to_call(kind):
    cache = Cache([9000, 3000], 2, 64, 64, kind, seed=3)
    q = torch.randn(2, 8 * 64).to(torch.bfloat16).cuda()
    outs = []
    for _ in range(5):
        outs.append(torch.empty_like(q))
        attention(cache, 8, q, outs[-1], i32([0, 1, 2]), i32([8999, 2999]), 1)
    assert all(torch.equal(o, outs[0]) for o in outs)


# ---- rules --------------------------------------------------------------------------------------------------------------------
def rules_exact(x, tokens, n_tokens, n_prompt, rep, pres, freq, bias, mask, mask_row):
    """fp32 one operation after the other, as the header states it (numpy rounds each)."""
    x = x.astype(np.float32).copy()
    rows, vocab = x.shape
    for r in range(rows):
        if tokens is not None:
            ids = tokens[r, :n_tokens[r]]
            ok = (ids >= 0) & (ids < vocab)
            said = np.arange(len(ids)) >= n_prompt[r]
            seen = np.unique(ids[ok])
            count = np.bincount(ids[ok & said], minlength=vocab)
            if rep is not None:
                x[r, seen] = np.where(x[r, seen] > 0, x[r, seen] / rep[r], x[r, seen] * rep[r])
            out = count > 0
            if freq is not None:
                x[r, out] -= freq[r] * count[out].astype(np.float32)
            if pres is not None:
                x[r, out] -= pres[r]
        if bias is not None:
            start, token, value = bias
            last = {int(token[i]): value[i] for i in range(start[r], start[r + 1])}
            for t, b in last.items():
                if 0 <= t < vocab:
                    x[r, t] = x[r, t] + b
        if mask is not None:
            m = r if mask_row is None else mask_row[r]
            if m >= 0:
                bits = (mask[m].astype(np.uint32)[:, None] >> np.arange(32, dtype=np.uint32) & 1).reshape(-1)[:vocab]
                x[r, bits == 0] = -np.inf
    return x


def check_rules(rows, vocab, history, dtype=torch.float32, pad=0, shift=0, penalties="rpf", biases=0, masks=0, by_row=True, in_place=False, seed=1,
                n_prompt=True):
    rng = np.random.default_rng(seed)
    ld = vocab + pad
    store = torch.from_numpy(rng.standard_normal((rows * ld + shift)).astype(np.float32) * 4).to(dtype).cuda()
    logits = store[shift:].view(rows, ld)[:, :vocab]
    out_store = torch.full((rows * ld + shift,), 7.0, device="cuda")
    out = logits if in_place else out_store[shift:].view(rows, ld)[:, :vocab]
    kw, host = {}, dict(tokens=None, n_tokens=None, n_prompt=None, rep=None, pres=None, freq=None, bias=None, mask=None, mask_row=None)
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    if history:
        tokens = np.minimum(rng.geometric(0.01, size=(rows, history)) * 7 - 7, vocab + 3).astype(np.int32)
        tokens[:, ::5] = rng.integers(0, vocab, size=tokens[:, ::5].shape)
        tokens[:, ::11] = -1
        n = rng.integers(0, history + 1, size=rows).astype(np.int32)
        n[0] = history
        prompt = (n // 2).astype(np.int32)
        host.update(tokens=tokens, n_tokens=n, n_prompt=prompt if n_prompt else 0 * prompt)
        kw.update(d_tokens=up(tokens), d_n_tokens=up(n), ld_tokens=history, d_n_prompt=up(prompt) if n_prompt else None)
        if "r" in penalties:
            host["rep"] = (1 + rng.random(rows)).astype(np.float32)
            kw["d_repetition"] = up(host["rep"])
        if "p" in penalties:
            host["pres"] = rng.random(rows).astype(np.float32)
            kw["d_presence"] = up(host["pres"])
        if "f" in penalties:
            host["freq"] = (rng.random(rows) - 0.3).astype(np.float32)
            kw["d_frequency"] = up(host["freq"])
    if biases:
        per = rng.integers(0, biases + 1, size=rows)
        per[-1] = biases
        start = np.concatenate([[3], 3 + np.cumsum(per)]).astype(np.int32)
        token = rng.integers(-2, vocab + 2, size=start[-1] + 1).astype(np.int32)
        token[start[-2]:start[-1]] = token[start[-2]]  # one row names one token again and again
        value = rng.standard_normal(token.size).astype(np.float32)
        value[::7] = -np.inf
        host["bias"] = (start, token, value)
        kw.update(d_bias_start=up(start), d_bias_token=up(token), d_bias=up(value))
    if masks:
        words = (vocab + 31) // 32 + 1
        m = masks if by_row else rows
        host["mask"] = rng.integers(0, 2 ** 32, size=(m, words), dtype=np.uint32)
        host["mask"][0] = 0  # nothing is allowed
        kw.update(d_mask=up(host["mask"].view(np.int32)), ld_mask=words, n_masks=m)
        if by_row:
            host["mask_row"] = rng.integers(-1, masks, size=rows).astype(np.int32)
            kw["d_mask_row"] = up(host["mask_row"])
    x = logits.float().cpu().numpy().copy()
    rules(logits, out, **kw)
    torch.cuda.synchronize()
    assert status() == 0
    want = rules_exact(x, **host)
    assert np.array_equal(out.cpu().numpy(), want)
    if not in_place:
        assert np.array_equal(logits.float().cpu().numpy(), x)
        rest = out_store[shift:].view(rows, ld)[:, vocab:]
        assert (rest == 7).all() and (out_store[:shift] == 7).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 1023), (3, 1024), (2, 4097), (64, 32000), (5, 50001), (130, 16385)])
def test_rules_match_their_definition(dtype, rows, vocab):
    check_rules(rows, vocab, 300, dtype, biases=40, masks=4)
    check_rules(rows, vocab, 300, dtype, biases=40, masks=4, pad=5, shift=3)


@pytest.mark.parametrize("kw", [
    dict(history=0), dict(history=0, masks=3), dict(history=0, masks=3, by_row=False), dict(history=0, biases=9), dict(history=1),
    dict(history=5000), dict(history=6000, biases=700), dict(history=12000, biases=700), dict(history=40000, biases=9), dict(history=200, penalties="r"), dict(history=200, penalties="p"), dict(history=200, penalties="f"),
    dict(history=200, penalties=""), dict(history=200, n_prompt=False), dict(history=200, biases=9, masks=2, in_place=True),
    dict(history=200, biases=9, masks=2, in_place=True, pad=3),
])
@pytest.mark.parametrize("rows", [2, 200])
def test_rules_one_by_one(rows, kw):
    check_rules(rows, 9001, **kw)


def test_rules_of_many_rows():
    check_rules(70000, 40, 3, biases=2, masks=2)
    check_rules(70000, 40, 3, masks=1, by_row=False)


def test_rules_masked_logits_may_be_anything():
    logits = torch.tensor([[math.nan, math.inf, -math.inf, 1.0, math.nan]], device="cuda")
    out = torch.empty_like(logits)
    rules(logits, out, d_mask=i32([[0b11000]]), ld_mask=1, n_masks=1)
    got = out.cpu()
    assert (got[0, :3] == -math.inf).all() and got[0, 3] == 1 and math.isnan(got[0, 4])


def test_rules_out_of_range_is_reported():
    logits = torch.randn(3, 100, device="cuda")
    out = torch.empty_like(logits)
    tokens = torch.zeros(3, 4, dtype=torch.int32, device="cuda")
    rep = torch.full((3,), 2.0, device="cuda")
    rules(logits, out, d_tokens=tokens, d_n_tokens=i32([4, 5, -1]), ld_tokens=4, d_repetition=rep)
    assert status() == BAD_INDEX
    assert torch.equal(out[1:], logits[1:]) and not torch.equal(out[0], logits[0])
    rules(logits, out, d_mask=i32([[0] * 4]), ld_mask=4, n_masks=1, d_mask_row=i32([1, -1, -1]))
    assert status() == BAD_INDEX and torch.equal(out, logits)
    rules(logits, out, d_bias_start=i32([0, 1, 0, 70000]), d_bias_token=i32([0, 0]), d_bias=rep)
    assert status() == BAD_INDEX and torch.equal(out[1:], logits[1:])


# ---- together -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", KINDS)
def test_one_captured_step_replayed_token_after_token(kind):
    """Append, attention, rules and the sampler as a captured step: places and token lists move on the device.  Another stream than the
    default one, and the same results as the calls one by one."""
    heads, kv, hd, page, seqs, vocab, steps = 8, 2, 64, 16, 3, 1000, 40
    cos, sin = rope_tables(128, hd)
    first = [5, 16, 40]
    g = torch.Generator().manual_seed(3)
    xs = torch.randn(steps, seqs, (heads + 2 * kv) * hd, generator=g).to(torch.bfloat16).cuda()
    head = torch.randn(vocab, heads * hd, generator=g).cuda()
    start = i32(starts([1] * seqs))
    rep = torch.full((seqs,), 1.5, device="cuda")
    mask = torch.randint(-2 ** 31, 2 ** 31 - 1, (1, 32), generator=g).to(torch.int32).cuda()
    mask_row = i32([0, -1, 0])

    def program(cache):
        s = {"qkv": torch.zeros_like(xs[0]), "q": torch.zeros(seqs, heads * hd, dtype=torch.bfloat16, device="cuda"), "pos": i32(first),
             "att": torch.zeros(seqs, heads * hd, dtype=torch.bfloat16, device="cuda"), "logits": torch.zeros(seqs, vocab, device="cuda"),
             "tokens": torch.zeros(seqs, steps, dtype=torch.int32, device="cuda"), "n": i32([0] * seqs), "work": workspace(heads, kv, hd)}

        def step(stream=None):
            append(cache, heads, s["qkv"], s["q"], start, s["pos"], cos, sin, stream=stream)
            attention(cache, heads, s["q"], s["att"], start, s["pos"], 1, work=s["work"], stream=stream)
            s["logits"].copy_(s["att"].float() @ head.T)
            rules(s["logits"], s["logits"], d_tokens=s["tokens"], d_n_tokens=s["n"], ld_tokens=steps, d_repetition=rep, d_mask=mask,
                  ld_mask=32, n_masks=1, d_mask_row=mask_row, stream=stream)
            s["tokens"].scatter_(1, s["n"][:, None].long(), s["logits"].argmax(1, keepdim=True).int())
            s["n"] += 1
            s["pos"] += 1

        return s, step

    def new_cache():
        return Cache([f + steps for f in first], kv, hd, page, kind, seed=8)

    one, step = program(new_cache())
    for t in range(steps):
        one["qkv"].copy_(xs[t])
        step()
    torch.cuda.synchronize()
    two, step = program(new_cache())
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        two["qkv"].copy_(xs[0])
        step(side.cuda_stream)  # warm-up: the matrix product's own set-up
    torch.cuda.synchronize()
    two, step = program(new_cache())
    graph = torch.cuda.CUDAGraph()
    keep = {k: v.clone() for k, v in two.items()}
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        step(side.cuda_stream)
    for k, v in keep.items():
        two[k].copy_(v)
    for t in range(steps):
        two["qkv"].copy_(xs[t])
        graph.replay()
    torch.cuda.synchronize()
    assert status() == 0
    assert torch.equal(one["tokens"], two["tokens"]) and torch.equal(one["logits"], two["logits"]) and torch.equal(one["att"], two["att"])
    assert len(set(one["tokens"].flatten().tolist())) > 10
    allowed = (mask[0].long()[one["tokens"][0].long() // 32] >> (one["tokens"][0].long() % 32)) & 1
    assert allowed.all()
    # the framework's sampler takes the same logits
    out = i32([0] * seqs)
    assert lib.ane_op_sample_rows(ptr(one["logits"]), None, 0.0, ptr(out), seqs, vocab) == 0
    assert torch.equal(out, one["logits"].argmax(1).int())
