"""The serving operators of the library, for timing them and for comparing them with their definitions.

One decoded token, or one piece of a prompt, takes three of them: `append` rotates the new queries and keys by their
positions and puts keys and values into a paged cache (ane_op_kv_append), `attend` lets the new queries look at the cache
(ane_op_kv_attention), `rules` applies penalties, biases and grammar masks to the logits before a token is drawn
(ane_op_logit_rules).  The cache holds bf16, or 8-bit floating point (e4m3) with one scale, a power of two, for each page and
head.  Head layouts are the ones of the benchmark's and the tests' models and generic ones; contexts go from a few tokens to
some ten thousand, vocabularies from 4096 to 128000.
"""
import ctypes
import math
import os
import sys

import torch

own = False

DEV = "cuda"
THETA = 10000.0
KV_BF16, KV_E4M3 = 0, 1
DTYPE_BF16, DTYPE_F32 = 0, 1

#: query heads, KV heads, head size
HEADS = {
    "small": (6, 6, 48), "middle": (8, 8, 64), "large": (12, 12, 64), "large_gqa": (12, 4, 64), "large_gqa6": (12, 6, 64),
    "narrow": (8, 1, 32), "wide": (32, 8, 128), "wide_mha": (8, 8, 128), "odd": (12, 4, 96), "shared": (16, 2, 128),
}


def _append(name, heads, seqs, new, past, page, cache):
    return {"name": name, "op": "append", "heads": heads, "seqs": seqs, "new": new, "past": past, "page": page, "cache": cache}


def _attend(name, heads, seqs, new, past, page, cache, window=0):
    return {"name": name, "op": "attend", "heads": heads, "seqs": seqs, "new": new, "past": past, "page": page, "cache": cache,
            "window": window}


def _rules(name, rows, vocab, history, masks, biases, logits):
    return {"name": name, "op": "rules", "rows": rows, "vocab": vocab, "history": history, "masks": masks, "biases": biases,
            "logits": logits}


def listed():
    return [
        # One interactive completion with the benchmark's model, in the middle of its window: latency alone counts.
        _append("append_1x1_bf16", "large", 1, 1, 200, 16, "bf16"),
        # A step of a serving batch: 64 sequences, a token each, grouped heads, 8-bit pages that are partly filled.
        _append("append_64x1_e4m3", "wide", 64, 1, 1000, 32, "e4m3"),
        # Prompts: ragged pieces of up to 512 tokens for 32 sequences, behind what their caches hold already.
        _append("append_32x512_e4m3", "large_gqa", 32, 512, 300, 64, "e4m3"),
        # One interactive completion: 12 heads, 256 tokens of context.
        _attend("attend_1x1_256_bf16", "large", 1, 1, 255, 16, "bf16"),
        # The generation workload of the benchmark: 32 sequences, grouped heads, up to 768 tokens.
        _attend("attend_32x1_768_bf16", "large_gqa", 32, 1, 767, 16, "bf16"),
        # A serving batch over long 8-bit caches of very different lengths.
        _attend("attend_64x1_8k_e4m3", "wide", 64, 1, 8000, 64, "e4m3"),
        # Two long documents with few KV heads: the keys have to be split over the whole chip.
        _attend("attend_2x1_60k_e4m3", "shared", 2, 1, 60001, 128, "e4m3"),
        # Drafted tokens checked in one go: up to five a sequence, small model with heads of 48.
        _attend("attend_16x5_500_bf16", "small", 16, 5, 500, 16, "bf16"),
        # A piece of a prompt against 8-bit pages: up to 400 queries a sequence behind up to 1500 tokens of context.
        _attend("attend_8x400_1500_e4m3", "large_gqa", 8, 400, 1500, 64, "e4m3"),
        # One completion: penalties for its 300 tokens, a few biases, no grammar.
        _rules("rules_1x32000", 1, 32000, 300, 0, 8, "f32"),
        # A serving batch: every rule, long histories, half of the rows under one of eight grammars' masks.
        _rules("rules_64x32000", 64, 32000, 2000, 8, 100, "f32"),
        # The largest vocabulary, bf16 logits, an odd number of rows.
        _rules("rules_255x128000_bf16", 255, 128000, 6000, 16, 300, "bf16"),
    ]


# ---- drawn cases ----------------------------------------------------------------------------------------------------
def _between(rng, lo, hi):
    """A whole number from lo to hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _padded(case):
    """Elements of K that a padded fp32 copy of the cache has, and scores."""
    h, kv, d = HEADS[case["heads"]]
    total = case["past"] + case["new"]
    return max(case["seqs"] * total * kv * d, case["seqs"] * case["new"] * total * h)


def draw(rng):
    op = rng.choice(["append", "append", "attend", "attend", "attend", "attend", "rules", "rules"])
    if op == "rules":
        rows, vocab = _between(rng, 1, 255), rng.choice([4096, 32000, 32000, 50001, 128000, _between(rng, 4096, 128000)])
        masks = rng.choice([0, 0, 1, _between(rng, 1, 16)])
        return {"op": op, "rows": rows, "vocab": vocab, "history": _between(rng, 1, 6000), "masks": masks,
                "biases": rng.choice([0, _between(rng, 1, 300)]), "logits": rng.choice(["f32", "f32", "bf16"])}
    case = {"op": op, "heads": rng.choice(sorted(HEADS)), "seqs": _between(rng, 1, 64), "new": 1, "past": 0,
            "page": rng.choice([16, 32, 64, 128]), "cache": rng.choice(["bf16", "e4m3"])}
    if op == "append":
        case["new"] = rng.choice([1, _between(rng, 1, 512)])
        case["past"] = _between(rng, 1, 1000)
        while case["seqs"] * case["new"] > 16384:
            case["seqs"] = (case["seqs"] + 1) // 2
        return case
    case["new"] = rng.choice([1, 1, _between(rng, 2, 8), _between(rng, 8, 400)])
    case["past"] = _between(rng, 1, 60000 if case["new"] <= 8 else 1500)
    case["window"] = rng.choice([0, 0, 0, _between(rng, 16, 4096)])
    while case["seqs"] > 1 and (_padded(case) > 64 * 8001 * 8 * 128 or work(case)["flops"] > 12e9):
        case["seqs"] = (case["seqs"] + 1) // 2
    return case


# ---- sizes ----------------------------------------------------------------------------------------------------------
def _spread(n, most, stride):
    """n lengths between a quarter of `most` and `most`, the first the longest."""
    return [max(1, most - (most * 3 // 4) * ((i * stride) % 101) // 101) for i in range(n)]


def _lengths(case):
    """New tokens and tokens that the cache holds before them, for each sequence."""
    return _spread(case["seqs"], case["new"], 37), _spread(case["seqs"], case["past"], 61)


def work(case):
    if case["op"] == "rules":
        rows, vocab = case["rows"], case["vocab"]
        history = sum(_spread(rows, case["history"], 53))
        size = 4 if case["logits"] == "f32" else 2
        moved = rows * vocab * (size + 4) + 4 * history + case["masks"] * ((vocab + 31) // 32) * 4 + rows * case["biases"] * 8
        return {"bytes": moved, "flops": rows * vocab}
    h, kv, d = HEADS[case["heads"]]
    size = 1 if case["cache"] == "e4m3" else 2
    new, past = _lengths(case)
    tokens = sum(new)
    if case["op"] == "append":
        # packed q|k|v in, the rotation of each position, rotated q and the cache's k and v out
        return {"bytes": tokens * (2 * (h + 2 * kv) * d + 4 * d + 2 * h * d + 2 * size * kv * d), "flops": 3 * tokens * (h + kv) * d}
    seen = pairs = 0
    for n, p in zip(new, past):
        window = case["window"] or p + n
        seen += p + n - max(0, p + 1 - window)
        pairs += sum(min(window, p + 1 + i) for i in range(n))
    return {"bytes": 2 * size * seen * kv * d + 4 * tokens * h * d, "flops": 4 * pairs * h * d}


# ---- what a user's program has in hand ------------------------------------------------------------------------------
def _paged(case, gen):
    """A cache with the tokens before this call, its page table and the sequences' places."""
    h, kv, d = HEADS[case["heads"]]
    new, past = _lengths(case)
    page, n = case["page"], case["seqs"]
    held = [(a + b + page - 1) // page for a, b in zip(new, past)]
    pages, pitch = sum(held) + 3, max(held)
    order = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
    table = torch.zeros(n, pitch, dtype=torch.int32)
    slots = torch.tensor([[sum(held[:b]) + min(i, held[b] - 1) for i in range(pitch)] for b in range(n)])
    table = order[slots.to(DEV)].contiguous()
    shape = (pages, kv, page, d)
    state = {"case": case, "table": table, "tokens": sum(new), "most_new": max(new), "n_pages": pages,
             "start": torch.tensor([0] + [sum(new[:b + 1]) for b in range(n)], dtype=torch.int32, device=DEV),
             "pos": torch.tensor(past, dtype=torch.int32, device=DEV)}
    for x in ("k", "v"):
        if case["cache"] == "bf16":
            state[x] = torch.randn(shape, generator=gen, device=DEV).to(torch.bfloat16)
            state[x + "_scale"] = None
        else:  # keys and values of about unit size, their pages filled to near the largest e4m3 value
            state[x] = (torch.randn(shape, generator=gen, device=DEV) * 100).clamp_(-448, 448).to(torch.float8_e4m3fn)
            state[x + "_scale"] = torch.exp2(torch.randint(-8, -5, (pages, kv), generator=gen, device=DEV).float())
    return state


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    if case["op"] == "rules":
        return _prepare_rules(case, gen)
    h, kv, d = HEADS[case["heads"]]
    state = _paged(case, gen)
    tokens = state["tokens"]
    if case["op"] == "append":
        # a few channels of keys are much larger than the others, as in trained models
        x = torch.randn(tokens, h + 2 * kv, d, generator=gen, device=DEV)
        x[:, h:h + kv] *= torch.exp(0.7 * torch.randn(kv, d, generator=gen, device=DEV))
        state["qkv"] = x.reshape(tokens, -1).to(torch.bfloat16)
        state["q"] = torch.empty(tokens, h * d, dtype=torch.bfloat16, device=DEV)
        most = case["new"] + case["past"]
        freq = THETA ** (-torch.arange(0, d, 2, dtype=torch.float64, device=DEV) / d)
        angle = torch.arange(most, dtype=torch.float64, device=DEV)[:, None] * freq
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
    else:
        state["q"] = (1.5 * torch.randn(tokens, h * d, generator=gen, device=DEV)).to(torch.bfloat16)
        state["out"] = torch.empty(tokens, h * d, dtype=torch.bfloat16, device=DEV)
    return state


def _prepare_rules(case, gen):
    rows, vocab, most = case["rows"], case["vocab"], case["history"]
    logits = 3 * torch.randn(rows, vocab, generator=gen, device=DEV)
    held = torch.tensor(_spread(rows, most, 53), dtype=torch.int32, device=DEV)
    # tokens of natural text come again and again: ranks with a density of 1 / rank
    tokens = torch.exp(torch.rand(rows, most, generator=gen, device=DEV) * math.log(vocab)).to(torch.int32) - 1
    state = {"case": case, "logits": logits.to(torch.bfloat16) if case["logits"] == "bf16" else logits,
             "tokens": tokens.clamp_(0, vocab - 1), "n_tokens": held, "n_prompt": held // 3,
             "repetition": 1 + 0.3 * torch.rand(rows, generator=gen, device=DEV),
             "presence": 0.5 * torch.rand(rows, generator=gen, device=DEV),
             "frequency": 0.2 * torch.rand(rows, generator=gen, device=DEV),
             "out": torch.empty(rows, vocab, device=DEV), "mask": None, "mask_row": None, "bias": None}
    if case["masks"]:
        words = (vocab + 31) // 32
        state["mask"] = torch.randint(-2 ** 31, 2 ** 31, (case["masks"], words), generator=gen, device=DEV, dtype=torch.int64).to(torch.int32)
        row = torch.randint(0, case["masks"], (rows,), generator=gen, device=DEV, dtype=torch.int32)
        state["mask_row"] = torch.where(torch.arange(rows, device=DEV) % 2 == 0, row, torch.full_like(row, -1))
    if case["biases"]:
        n = case["biases"]
        state["bias_start"] = torch.arange(rows + 1, dtype=torch.int32, device=DEV) * n
        first = torch.randint(0, vocab, (rows, 1), generator=gen, device=DEV)
        state["bias_token"] = ((first + torch.arange(n, device=DEV) * (vocab // n)) % vocab).to(torch.int32).reshape(-1)
        state["bias"] = 2 * torch.randn(rows * n, generator=gen, device=DEV)
    return state


# ---- the definitions in elementary operations -----------------------------------------------------------------------
def _where(s):
    """The sequence and the position of every new token."""
    at = torch.arange(s["tokens"], dtype=torch.int32, device=DEV)
    seq = torch.searchsorted(s["start"][1:], at, right=True)
    return seq, (s["pos"][seq] + at - s["start"][seq]).long()


def _power_of_two(largest):
    """The smallest power of two, at least 2^-126, that brings values of this size within 448."""
    m, e = torch.frexp(largest.double() / 448)
    e = torch.where(m == 0.5, e - 1, e)
    return torch.exp2(torch.where(largest > 0, e, -126).clamp(min=-126).double()).float()


def _put_8bit(s, name, x, seq, pos):
    """New rows x [tokens, KV, hd] into 8-bit pages: a page's scale grows to hold them, and its older rows follow."""
    cache, scale, page, table = s[name], s[name + "_scale"], s["case"]["page"], s["table"].long()
    raw = cache.view(torch.uint8)
    at, off = table[seq, pos // page], pos % page
    top = torch.zeros_like(scale).scatter_reduce_(0, at[:, None].expand(-1, scale.shape[1]), x.abs().amax(-1), "amax")
    fresh = torch.zeros_like(scale[:, 0]).index_add_(0, at, (off == 0).float()) > 0
    touched = torch.zeros_like(fresh).index_fill_(0, at, True)
    old = torch.where(fresh[:, None], 0.0, scale)
    now = torch.where(touched[:, None], torch.maximum(old, _power_of_two(top)), scale)
    held = s["pos"].long() % page
    first = table.gather(1, (s["pos"].long() // page)[:, None])[:, 0]
    ratio = (scale / now)[first][:, :, None, None]
    moved = (cache[first].float() * ratio).to(torch.float8_e4m3fn).view(torch.uint8)
    keep = (torch.arange(page, device=DEV)[None] < held[:, None])[:, None, :, None]
    raw[first] = torch.where(keep, moved, raw[first])
    raw[at, :, off] = (x / now[at][:, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    scale.copy_(now)


def _put_bf16(s, name, x, seq, pos):
    page = s["case"]["page"]
    s[name][s["table"].long()[seq, pos // page], :, pos % page] = x.to(torch.bfloat16)


def _append_plain(s):
    case = s["case"]
    h, kv, d = HEADS[case["heads"]]
    seq, pos = _where(s)
    x = s["qkv"].view(-1, h + 2 * kv, d).float()
    even, odd = x[:, :h + kv, 0::2], x[:, :h + kv, 1::2]
    c, n = s["cos"][pos][:, None], s["sin"][pos][:, None]
    turned = torch.stack([even * c - odd * n, odd * c + even * n], -1).flatten(-2)
    q = turned[:, :h].reshape(-1, h * d).to(torch.bfloat16)
    put = _put_8bit if case["cache"] == "e4m3" else _put_bf16
    put(s, "k", turned[:, h:], seq, pos)
    put(s, "v", x[:, h + kv:], seq, pos)
    return q


def _attend_plain(s):
    case = s["case"]
    h, kv, d = HEADS[case["heads"]]
    n, most, ids = case["seqs"], s["most_new"], s["table"].long()

    def dense(name):  # [n, kv, positions, d]
        x = s[name][ids].float()
        if s[name + "_scale"] is not None:
            x = x * s[name + "_scale"][ids][..., None, None]
        return x.transpose(1, 2).reshape(n, kv, -1, d)

    at = torch.arange(most, device=DEV)
    row = (s["start"][:-1, None] + at).clamp(max=s["tokens"] - 1).long()
    q = s["q"][row].view(n, most, kv, h // kv, d).float().permute(0, 2, 1, 3, 4).reshape(n, kv, -1, d)
    k = dense("k")
    scores = q @ k.transpose(2, 3)
    scores = (scores * d ** -0.5).view(n, kv, most, h // kv, -1)
    mine = (s["pos"][:, None] + at)[:, None, :, None, None]
    theirs = torch.arange(k.shape[2], device=DEV)
    del k
    seen = theirs <= mine
    if case["window"]:
        seen = seen & (theirs > mine - case["window"])
    scores = torch.where(seen, scores, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = p.view(n, kv, -1, p.shape[-1]) @ dense("v")
    out = out.view(n, kv, most, h // kv, d).permute(0, 2, 1, 3, 4).reshape(n, most, h * d)
    seq, pos = _where(s)
    return out[seq, pos - s["pos"][seq]].to(torch.bfloat16)


def _rules_plain(s):
    x = s["logits"].float()
    rows, vocab = x.shape
    at = torch.arange(s["tokens"].shape[1], device=DEV)
    said = at >= s["n_prompt"][:, None]
    known = at < s["n_tokens"][:, None]
    ids = s["tokens"].long()
    count = torch.zeros(rows, vocab + 1, device=DEV)
    count.scatter_add_(1, torch.where(known & said, ids, vocab), torch.ones_like(ids, dtype=torch.float32))
    seen = torch.zeros(rows, vocab + 1, dtype=torch.bool, device=DEV).scatter_(1, torch.where(known, ids, vocab), True)
    count, seen = count[:, :vocab], seen[:, :vocab]
    r = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * count
    x = x - torch.where(count > 0, s["presence"][:, None], 0.0)
    if s["bias"] is not None:
        row = torch.searchsorted(s["bias_start"][1:], torch.arange(s["bias"].numel(), dtype=torch.int32, device=DEV), right=True)
        token = s["bias_token"].long()
        x[row, token] = x[row, token] + s["bias"]
    if s["mask"] is not None:
        bits = (s["mask"][:, :, None] >> torch.arange(32, dtype=torch.int32, device=DEV)) & 1
        bits = bits.flatten(1)[:, :vocab].bool()
        free = s["mask_row"][:, None] < 0
        x = torch.where(bits[s["mask_row"].clamp(min=0).long()] | free, x, -math.inf)
    return x


# ---- the library's calls --------------------------------------------------------------------------------------------
def _calls(s):
    """The argument structures that a program fills in once for its buffers, and the call."""
    package = os.path.join(os.getcwd(), "autoresearch-go-ane_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    from ane import _ffi

    case, p = s["case"], lambda name: s[name].data_ptr() if s.get(name) is not None else None  # noqa: E731
    if case["op"] == "rules":
        a = _ffi.LogitRulesArgs(
            struct_size=ctypes.sizeof(_ffi.LogitRulesArgs), dtype=DTYPE_F32 if case["logits"] == "f32" else DTYPE_BF16,
            d_logits=p("logits"), d_out=p("out"), ld_logits=case["vocab"], ld_out=case["vocab"], rows=case["rows"],
            vocab=case["vocab"], d_tokens=p("tokens"), d_n_tokens=p("n_tokens"), d_n_prompt=p("n_prompt"),
            ld_tokens=case["history"], n_masks=case["masks"], d_mask=p("mask"), d_mask_row=p("mask_row"),
            ld_mask=(case["vocab"] + 31) // 32, d_bias_start=p("bias_start"), d_bias_token=p("bias_token"), d_bias=p("bias"),
            d_repetition=p("repetition"), d_presence=p("presence"), d_frequency=p("frequency"))
        return _ffi.lib.ane_op_logit_rules, ctypes.byref(a), (a,)
    h, kv, d = HEADS[case["heads"]]
    cache = _ffi.KvCache(
        struct_size=ctypes.sizeof(_ffi.KvCache), dtype=KV_E4M3 if case["cache"] == "e4m3" else KV_BF16, d_k=p("k"), d_v=p("v"),
        d_k_scale=p("k_scale"), d_v_scale=p("v_scale"), page_stride=0, n_pages=s["n_pages"], page_size=case["page"],
        n_kv_heads=kv, head_dim=d, d_page_table=p("table"), table_pitch=s["table"].shape[1])
    if case["op"] == "append":
        a = _ffi.KvAppendArgs(
            struct_size=ctypes.sizeof(_ffi.KvAppendArgs), n_heads=h, cache=ctypes.pointer(cache), d_qkv=p("qkv"), d_q=p("q"),
            ld_qkv=(h + 2 * kv) * d, ld_q=h * d, d_cos=p("cos"), d_sin=p("sin"), n_positions=s["cos"].shape[0],
            n_seq=case["seqs"], d_seq_start=p("start"), d_pos=p("pos"), n_tokens=s["tokens"])
        return _ffi.lib.ane_op_kv_append, ctypes.byref(a), (a, cache)
    room = _ffi.lib.ane_op_kv_attention_workspace(h, kv, d)
    s["workspace"] = torch.empty(room, dtype=torch.uint8, device=DEV)
    a = _ffi.KvAttentionArgs(
        struct_size=ctypes.sizeof(_ffi.KvAttentionArgs), n_heads=h, cache=ctypes.pointer(cache), d_q=p("q"), d_out=p("out"),
        ld_q=h * d, ld_out=h * d, d_seq_start=p("start"), d_pos=p("pos"), n_seq=case["seqs"], n_tokens=s["tokens"],
        max_new=s["most_new"], window=case["window"], scale=0.0, d_workspace=p("workspace"), workspace_bytes=room)
    return _ffi.lib.ane_op_kv_attention, ctypes.byref(a), (a, cache)


def run(state):
    op = state["case"]["op"]
    if own:
        if "call" not in state:
            state["call"] = _calls(state)
        call, args, _ = state["call"]
        if call(args) != 0:
            raise RuntimeError("the call was refused")
        got = state["q"] if op == "append" else state["out"]
    else:
        got = {"append": _append_plain, "attend": _attend_plain, "rules": _rules_plain}[op](state)
    if op != "append":
        return got
    if state["k_scale"] is None:
        return [got, state["k"], state["v"]]
    return [got, state["k"], state["v"], state["k_scale"], state["v_scale"]]


# ---- the same from the definitions in 64 bits -----------------------------------------------------------------------
def _exact_append(s):
    case = s["case"]
    h, kv, d = HEADS[case["heads"]]
    new, past = _lengths(case)
    page, kept = case["page"], {}
    table = s["table"].cpu()
    x = s["qkv"].double().view(-1, h + 2 * kv, d)
    pos = torch.cat([torch.arange(p, p + n) for n, p in zip(new, past)]).to(DEV)
    pair = torch.view_as_complex(x[:, :h + kv].reshape(-1, h + kv, d // 2, 2).contiguous())
    # the rotation is the caller's table, taken as it is
    turn = torch.complex(s["cos"][pos].double(), s["sin"][pos].double())
    turned = torch.view_as_real(pair * turn[:, None]).flatten(-2)
    for name, rows in (("k", turned[:, h:]), ("v", x[:, h + kv:])):
        values, first = s[name].double(), 0
        scale = None if s[name + "_scale"] is None else s[name + "_scale"].double()
        for b, (n, p) in enumerate(zip(new, past)):
            for slot in range(p // page, (p + n - 1) // page + 1):
                lo, hi, at = max(p, slot * page), min(p + n, (slot + 1) * page), int(table[b, slot])
                part = rows[first + lo - p:first + hi - p].transpose(0, 1)
                if scale is None:
                    values[at, :, lo - slot * page:hi - slot * page] = part
                    continue
                need = torch.exp2(torch.ceil(torch.log2(part.abs().amax((1, 2)) / 448)).clamp(min=-126))
                was = scale[at].clone()
                scale[at] = need if lo == slot * page else torch.maximum(was, need)
                if lo > slot * page:
                    values[at, :, :lo - slot * page] *= (was / scale[at])[:, None, None]
                values[at, :, lo - slot * page:hi - slot * page] = part / scale[at][:, None, None]
            first += n
        kept[name], kept[name + "_scale"] = values, scale
    got = [turned[:, :h].reshape(-1, h * d), kept["k"], kept["v"]]
    return got if kept["k_scale"] is None else got + [kept["k_scale"], kept["v_scale"]]


def _exact_attend(s):
    case = s["case"]
    h, kv, d = HEADS[case["heads"]]
    new, past = _lengths(case)
    out, first = torch.empty(s["tokens"], h, d, dtype=torch.float64, device=DEV), 0
    for b, (n, p) in enumerate(zip(new, past)):
        blocks = s["table"][b, :(p + n + case["page"] - 1) // case["page"]].long()
        for g in range(kv):
            def held(name):
                x = s[name][blocks, g].double()
                if s[name + "_scale"] is not None:
                    x *= s[name + "_scale"][blocks, g].double()[:, None, None]
                return x.reshape(-1, d)[:p + n]

            k, v = held("k"), held("v")
            away = (p + torch.arange(n, device=DEV))[:, None] - torch.arange(p + n, device=DEV)
            hidden = away < 0
            if case["window"]:
                hidden |= away >= case["window"]
            heads = range(g * (h // kv), (g + 1) * (h // kv))
            for j in heads:
                q = s["q"].view(-1, h, d)[first:first + n, j].double()
                scores = (q @ k.T / math.sqrt(d)).masked_fill_(hidden, -math.inf)
                out[first:first + n, j] = torch.softmax(scores, -1) @ v
        first += n
    return out.view(-1, h * d)


def _exact_rules(s):
    case = s["case"]
    x = s["logits"].double()
    rows, vocab = x.shape
    at = torch.arange(vocab, device=DEV)
    for r, held in enumerate(_spread(rows, case["history"], 53)):
        ids = s["tokens"][r, :held].long()
        count = torch.bincount(ids[held // 3:], minlength=vocab).double()
        seen = torch.bincount(ids, minlength=vocab) > 0
        by = s["repetition"][r].double()
        x[r, seen] = torch.where(x[r, seen] > 0, x[r, seen] / by, x[r, seen] * by)
        x[r] -= s["frequency"][r].double() * count + s["presence"][r].double() * (count > 0)
        if s["bias"] is not None:
            mine = slice(r * case["biases"], (r + 1) * case["biases"])
            x[r].index_add_(0, s["bias_token"][mine].long(), s["bias"][mine].double())
        if s["mask"] is not None and int(s["mask_row"][r]) >= 0:
            word = s["mask"][int(s["mask_row"][r])].long()[at // 32]
            x[r].masked_fill_(((word >> (at % 32)) & 1) == 0, -math.inf)
    return x


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "rules": _exact_rules}[case["op"]](s)
