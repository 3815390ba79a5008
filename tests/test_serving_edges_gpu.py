"""Serving operators where their inputs are legal but far from ordinary: scales that differ by powers of two without end, hidden pages, draws
at the ends of their range, places that nothing fits."""
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch
from oracle import oracle as O
from serving_utils import (BAD_INDEX, Cache, append, attention, attention_exact, attention_tolerance, i32, lib, ptr, rope_tables, rules, starts,
                           status)
from test_generate_gpu import CLEAR, forward, pair
from test_serving_gpu import KINDS, check_attention, qkv_rows

pytestmark = pytest.mark.gpu


# ---- scales of values -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("new", [1, 4, 40, 100])
@pytest.mark.parametrize("window", [0, 70])
def test_attention_scales_of_pages_that_a_row_does_not_see(page, new, window):
    """Values 2^30 times the others', ahead of all rows but the last ones and, with a window, behind all but the first ones."""
    pos = 200
    cache = Cache([pos + new], 2, 64, page, "e4m3", seed=4)
    loud = {(pos + new - 1) // page} if new > 1 else set()
    if window:
        loud.add((pos + 1 - window) // page)
    for slot in loud:
        cache.vs[cache.table_host[0][slot]] *= 2.0 ** 30
    check_attention("e4m3", 4, 2, 64, page, [new], [pos], window=window, cache=cache)


@pytest.mark.parametrize("new", [1, 8, 100])
@pytest.mark.parametrize("ratio", [26, 30, 36, 100])
@pytest.mark.parametrize("first", [True, False])
def test_attention_concentrated_on_pages_of_small_scales(new, ratio, first):
    """A row whose probabilities lie on pages with values far smaller than those of others that it sees: 48 in the exponent less there, or 96 where
    the values differ by more than that outweighs."""
    heads, kv, hd, page, pos = 2, 1, 64, 16, 300
    n = pos + new
    cache = Cache([n], kv, hd, page, "e4m3", seed=6)
    sign = torch.where(torch.rand(hd, generator=torch.Generator().manual_seed(1)) < 0.5, -1.0, 1.0)
    # scores are 64 * 0.25 * 8^-1 = 2 times a key's size: 0 and 0.875 on ordinary pages
    size = torch.where(torch.rand(n, generator=torch.Generator().manual_seed(2)) < 0.5, 0.0, 0.4375)
    large = range(0, 6) if first else range(10, 16)
    for slot in large:
        size[slot * page:(slot + 1) * page] = -24.0 if ratio < 60 else -48.0
        cache.vs[cache.table_host[0][slot]] *= 2.0 ** ratio
    cache.ks.fill_(1.0)
    rows = (size[:, None] * sign).to(torch.float8_e4m3fn)
    for p in range(n):
        cache.k[cache.table_host[0][p // page], (p % page) * hd:(p % page + 1) * hd] = rows[p].cuda()
    q = (0.25 * sign).repeat(new, heads).to(torch.bfloat16).cuda()
    out = torch.full_like(q, 7.0)
    attention(cache, heads, q, out, i32([0, new]), i32([pos]), new)
    assert status() == 0
    k, v = cache.rows("k", 0, n), cache.rows("v", 0, n)
    mq = q.double().cpu().view(new, heads, hd)
    ref, mass, big = attention_exact(mq, k, v, pos, hd ** -0.5, 0)
    tol = attention_tolerance(ref, mass, big, "e4m3", hd, n, mq, hd ** -0.5, float(k.abs().max()))
    got = out.double().cpu().view(new, heads, hd)
    assert ((got - ref).abs() <= tol).all(), float((got - ref).norm() / ref.norm())


# ---- probabilities --------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", [32, 48, 64, 96, 128])
@pytest.mark.parametrize("new", [1, 12, 90])
def test_attention_is_as_exact_with_many_rows_as_with_few(kind, hd, new):
    """What is left of the error is the result's rounding: probabilities enter with errors of 2^-16 (bf16 with a rest) or 2^-12 (f16), against 2^-8 at
    most, so that the error's norm exceeds the rounding's by less than one in a hundred; a twentieth is granted."""
    heads, kv, pos = 4, 2, 300
    cache, q, out = check_attention(kind, heads, kv, hd, 64, [new], [pos], loud=2.0)
    k, v = cache.rows("k", 0, pos + new), cache.rows("v", 0, pos + new)
    ref, _, _ = attention_exact(q.double().cpu().view(new, heads, hd), k, v, pos, hd ** -0.5, 0)
    off = (out.double().cpu().view(new, heads, hd) - ref).norm()
    rounding = (ref.to(torch.bfloat16).double() - ref).norm()
    assert off <= 1.05 * rounding, float(off / rounding)


# ---- draws among masked logits --------------------------------------------------------------------------------------------------
ENDS = [0.0, 5e-324, 2.0 ** -60, 1.0 - 2.0 ** -53]


def sample(logits, u, temperature):
    out = torch.full((logits.shape[0],), -7, dtype=torch.int32, device="cuda")
    assert lib.ane_op_sample_rows(ptr(logits), ptr(u), temperature, ptr(out), *logits.shape) == 0, lib.ane_ops_last_error()
    return out.cpu().numpy()


@pytest.mark.parametrize("temperature", [0.3, 1.0, 7.0])
@pytest.mark.parametrize("vocab,away", [(2, [0]), (2, [1]), (7, [0, 6]), (600, [0, 1, 2, 3, 597, 598, 599]), (32000, [*range(300), 5000, *range(31500, 32000)])])
def test_sampler_does_not_draw_what_a_mask_forbids(vocab, away, temperature):
    """Rules and then the sampler, with draws at both ends: the first and the last token with weight, and no token without."""
    rng = np.random.default_rng(3)
    x = torch.from_numpy((3 * rng.standard_normal((len(ENDS) + 20, vocab))).astype(np.float32)).cuda()
    u = np.concatenate([ENDS, rng.random(20)])
    words = np.full((vocab + 31) // 32, 0xffffffff, dtype=np.uint32)
    for v in away:
        words[v // 32] &= ~np.uint32(1 << v % 32)
    rules(x, x, d_mask=torch.from_numpy(words.view(np.int32)).cuda(), ld_mask=len(words), n_masks=1, d_mask_row=i32([0] * len(u)))
    got = sample(x, torch.from_numpy(u).cuda(), temperature)
    may = np.setdiff1d(np.arange(vocab), away)
    assert np.isin(got, may).all(), got
    assert got[0] == may[0] and got[1] == may[0]
    assert got[3] == may[-1] or vocab > 7  # the last token's weight may be below the draw's distance from 1


def test_sampler_without_masks_draws_what_it_drew():
    x = torch.full((5, 1000), 0.5, device="cuda")
    x[4] = math.nan
    got = sample(x, torch.tensor([0.0, 1e-300, 0.5, 1.0 - 2.0 ** -53, 0.5], dtype=torch.float64, device="cuda"), 1.0)
    assert got.tolist() == [0, 0, 499, 999, 999]


@pytest.mark.parametrize("kv", KINDS)
def test_generate_draws_allowed_tokens_only(kv):
    cfg, e = pair(vocab=512)
    allowed = np.random.default_rng(4).random(cfg["vocab"]) < 0.4
    allowed[[0, 1, cfg["vocab"] - 1]] = False
    prompts = [O.zipf_tokens(n, cfg["vocab"], n) for n in (40, 3, 17)]
    for end in ENDS:
        got = e.generate(prompts, 12, kv=kv, temperature=1.0, uniforms=np.full((12, 3), end), allowed=allowed)
        assert allowed[got].all(), (end, got)
    # without a mask, a draw of 0 is the first token
    got = e.generate(prompts, 6, kv=kv, temperature=1.0, uniforms=np.zeros((6, 3)), bias={7: 5.0})
    assert (got == 0).all()
    e.close()


# ---- places that nothing fits ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new,pos", [([1, 1, 1], [18, 19, 20]), ([15], [10]), ([3], [16]), ([30, 2], [0, 25]), ([40, 1], [15, 19])])
def test_append_behind_the_rotation_tables_is_not_written(kind, new, pos):
    """Tables of 20 positions, a cache of more: what lies within them is appended as if the other tokens were not there, which leave queries, keys,
    values and scales as they are."""
    heads, kv, hd, page, n_positions = 4, 2, 64, 16, 20
    cos, sin = rope_tables(n_positions, hd)
    start = starts(new)
    qkv = qkv_rows(start[-1], heads, kv, hd, 3)
    fits = [max(0, min(n, n_positions - p)) for n, p in zip(new, pos)]
    results = []
    for lens in (new, fits):
        cache = Cache([60, 60, 60][:len(new)], kv, hd, page, kind, seed=2)
        q = torch.full((start[-1], heads * hd), 7.0, dtype=torch.bfloat16, device="cuda")
        if lens is new:
            append(cache, heads, qkv, q, i32(start), i32(pos), cos, sin)
        else:
            for b, n in enumerate(fits):  # one sequence after the other: their rows are not next to one another
                if n == 0:
                    continue
                one = Cache([60, 60, 60][:len(new)], kv, hd, page, kind, seed=2)
                one.k, one.v, one.ks, one.vs, one.table = cache.k, cache.v, cache.ks, cache.vs, cache.table[b:b + 1].contiguous()
                rows = slice(start[b], start[b] + n)
                append(one, heads, qkv[rows], q[rows], i32([0, n]), i32([pos[b]]), cos, sin)
        assert status() == (BAD_INDEX if lens is new and fits != new else 0)  # 16 .. 18 fit
        results.append([q, cache.k.view(torch.uint8), cache.v.view(torch.uint8)] + ([cache.ks, cache.vs] if kind == "e4m3" else []))
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("kind", KINDS)
def test_attention_of_rows_that_many_sequences_claim_is_refused(kind):
    """Starts that go up and down give every second sequence the same 400 rows: more work than the tokens that the host knows of can be, which is
    what keeps the line of all tiles within 32 bits."""
    heads, kv, hd, rows, seqs = 4, 1, 64, 400, 2001
    cache = Cache([600], kv, hd, 64, kind, seed=5)
    cache.table = cache.table.expand(seqs, -1).contiguous()
    q = torch.randn(rows, heads * hd, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16).cuda()
    out = torch.full_like(q, 7.0)
    start = i32([rows * (b % 2) for b in range(seqs + 1)])
    attention(cache, heads, q, out, start, i32([100] * seqs), rows)
    assert status() == BAD_INDEX and (out == 7).all()
    # as many sequences that do not
    attention(cache, heads, q, out, i32([min(b, rows) for b in range(seqs + 1)]), i32([100] * seqs), rows)
    assert status() == 0 and not (out == 7).all(1).any()


FIRST_CALLS = """
import sys, threading
sys.path[:0] = sys.argv[1:]
import conftest, torch
from serving_utils import Cache, attention_args, i32, lib, status, workspace, BAD_INDEX
import ctypes
cache = Cache([32], 1, 64, 16, "bf16")
q = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
out, work = torch.zeros_like(q), workspace(1, 1, 64)
start, pos = i32([0, 4]), i32([-3])
streams = [torch.cuda.Stream() for _ in range(8)]
args = [attention_args(cache, 1, q, out, start, pos, 4, work=torch.empty_like(work), stream=s.cuda_stream) for s in streams]
torch.cuda.synchronize()
torch.cuda._sleep(200_000_000)  # the default stream is busy for a tenth of a second
threads = [threading.Thread(target=lambda a=a: lib.ane_op_kv_attention(ctypes.byref(a))) for a in args]
for t in threads: t.start()
for t in threads: t.join()
for s in streams: s.synchronize()
assert status() == BAD_INDEX
assert status() == 0
"""


def test_first_calls_on_busy_devices_and_several_threads_keep_their_reports():
    """The status word is taken by the first call of a process: on streams that do not wait for the default one, while that one is busy."""
    here = os.path.dirname(os.path.abspath(__file__))
    root = os.path.dirname(here)
    run = subprocess.run([sys.executable, "-c", FIRST_CALLS, here, root, os.path.join(root, "autoresearch-go-ane_b200")], capture_output=True, text=True,
                         timeout=300, env=dict(os.environ, CUDA_MODULE_LOADING="EAGER"))  # else the first launch waits for the device
    assert run.returncode == 0, run.stderr[-2000:]


# ---- generation of many prompts at once -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("kv", KINDS)
def test_generate_of_forty_ragged_prompts_gives_what_each_gives_alone(kv):
    """More sequences than the dense kernels take.  Each row follows from its own prompt: a token is the best one of a full forward pass but for what
    bf16 (the margin of the other tests) or 8-bit caches can turn round, and what its prompt gives alone up to the first place where two tokens are
    as near as that."""
    cfg, e = pair(batch=40, seq=100, layers=2)
    prompts = [O.zipf_tokens(1 + 2 * b, cfg["vocab"], b) for b in range(40)]
    got = e.generate(prompts, 21, kv=kv)
    same = 0
    for b, p in enumerate(prompts):
        alone = e.generate([p], 21, kv=kv)[0]
        apart = False
        for i, col in enumerate(forward(e, cfg, p, got[b])):
            near = CLEAR if kv == "bf16" else 0.5 * float(col.std())
            assert col.max() - col[got[b, i]] <= near, (b, i)
            apart = apart or got[b, i] != alone[i]
            if apart:
                assert abs(col[got[b, i]] - col[alone[i]]) <= near, (b, i)
                break
            same += 1
    assert same > 40 * 21 // 2, same
    assert len({tuple(r) for r in got.tolist()}) > 20  # prompts lead to different texts
    e.close()
