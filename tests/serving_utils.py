"""What the tests of the serving operators share: a paged cache on the GPU, the calls, and their definitions in 64 bits."""
import ctypes
import math

import numpy as np
import torch
from ane import _ffi

lib = _ffi.lib
BAD_INDEX = 110


def ptr(t):
    return None if t is None else t.data_ptr()


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def status():
    v = ctypes.c_int32(0)
    assert lib.ane_ops_device_status(ctypes.byref(v)) == 0
    return v.value


def e4m3(x):
    return x.to(torch.float8_e4m3fn)


class Cache:
    """Pages in random order; `extra`: elements between pages that belong to nobody (they must stay as they are)."""

    def __init__(self, room, kv, hd, page, kind, seed=0, extra=0, spare=3, fill=True):
        g = torch.Generator().manual_seed(seed)
        held = [max(1, -(-r // page)) for r in room]
        self.kv, self.hd, self.page, self.kind, self.pages = kv, hd, page, kind, sum(held) + spare
        self.pitch = max(held) + 1
        order = torch.randperm(self.pages, generator=g).tolist()
        table, at = [], 0
        for n in held:  # entries that no token needs point nowhere
            table.append([order[at + i] if i < n else -7 for i in range(self.pitch)])
            at += n
        self.table_host = table
        self.table = i32(table)
        self.stride = kv * page * hd + extra
        dt = torch.bfloat16 if kind == "bf16" else torch.float8_e4m3fn
        shape = (self.pages, self.stride)
        if fill:
            raw = [torch.randn(shape, generator=g) * (1 if kind == "bf16" else 90) for _ in range(2)]
            self.k, self.v = (x.clamp(-448, 448).to(dt).cuda() for x in raw)
        else:
            self.k, self.v = (torch.zeros(shape, dtype=torch.uint8, device="cuda").view(dt) if kind != "bf16" else
                              torch.zeros(shape, dtype=dt, device="cuda") for _ in range(2))
        self.ks = self.vs = None
        if kind != "bf16":
            self.ks, self.vs = (torch.exp2(torch.randint(-8, -5, (self.pages, kv), generator=g).float()).cuda() for _ in range(2))

    def struct(self, **over):
        c = _ffi.KvCache(struct_size=ctypes.sizeof(_ffi.KvCache), dtype=_ffi.KV_BF16 if self.kind == "bf16" else _ffi.KV_E4M3,
                         d_k=ptr(self.k), d_v=ptr(self.v), d_k_scale=ptr(self.ks), d_v_scale=ptr(self.vs),
                         page_stride=self.stride, n_pages=self.pages, page_size=self.page, n_kv_heads=self.kv, head_dim=self.hd,
                         d_page_table=ptr(self.table), table_pitch=self.pitch)
        for k, v in over.items():
            setattr(c, k, v)
        return c

    def blocks(self, x):  # [pages, kv, page, hd] of a raw buffer
        return x[:, :self.kv * self.page * self.hd].reshape(self.pages, self.kv, self.page, self.hd)

    def values(self, name):  # what the cache stands for, in 64 bits, on the CPU
        x = self.blocks(getattr(self, name)).cpu()
        s = self.ks if name == "k" else self.vs
        x = x.float().double()
        return x if s is None else x * s.cpu().double()[..., None, None]

    def rows(self, name, b, n):  # [n, kv, hd] of sequence b
        v = self.values(name)
        return torch.stack([v[self.table_host[b][p // self.page], :, p % self.page] for p in range(n)]) if n else \
            torch.zeros(0, self.kv, self.hd, dtype=torch.float64)


def starts(new, before=0):
    return [before + sum(new[:b]) for b in range(len(new) + 1)]


def append_args(cache, heads, qkv, q, start, pos, cos, sin, n_tokens=None, stream=None, **over):
    c = cache.struct()
    a = _ffi.KvAppendArgs(struct_size=ctypes.sizeof(_ffi.KvAppendArgs), n_heads=heads, cache=ctypes.pointer(c), d_qkv=ptr(qkv),
                          d_q=ptr(q), ld_qkv=qkv.stride(0), ld_q=0 if q is None else q.stride(0), d_cos=ptr(cos), d_sin=ptr(sin),
                          n_positions=0 if cos is None else cos.shape[0], n_seq=start.numel() - 1, d_seq_start=ptr(start),
                          d_pos=ptr(pos), n_tokens=qkv.shape[0] if n_tokens is None else n_tokens, stream=stream)
    for k, v in over.items():
        setattr(a, k, v)
    a.keep = c
    return a


def append(*args, **kw):
    a = append_args(*args, **kw)
    rc = lib.ane_op_kv_append(ctypes.byref(a))
    assert rc == 0, lib.ane_ops_last_error()


def workspace(heads, kv, hd):
    n = lib.ane_op_kv_attention_workspace(heads, kv, hd)
    assert n > 0
    return torch.full((n,), 0xff, dtype=torch.uint8, device="cuda")  # NaN wherever it is read before it is written


def attention_args(cache, heads, q, out, start, pos, max_new, window=0, scale=0.0, work=None, stream=None, **over):
    c = cache.struct()
    work = workspace(heads, cache.kv, cache.hd) if work is None else work
    a = _ffi.KvAttentionArgs(struct_size=ctypes.sizeof(_ffi.KvAttentionArgs), n_heads=heads, cache=ctypes.pointer(c), d_q=ptr(q),
                             d_out=ptr(out), ld_q=q.stride(0), ld_out=out.stride(0), d_seq_start=ptr(start), d_pos=ptr(pos),
                             n_seq=start.numel() - 1, n_tokens=q.shape[0], max_new=max_new, window=window, scale=scale,
                             d_workspace=ptr(work), workspace_bytes=work.numel(), stream=stream)
    for k, v in over.items():
        setattr(a, k, v)
    a.keep = (c, work)
    return a


def attention(*args, **kw):
    a = attention_args(*args, **kw)
    rc = lib.ane_op_kv_attention(ctypes.byref(a))
    assert rc == 0, lib.ane_ops_last_error()


def rope_tables(n, hd, theta=10000.0):
    at = torch.arange(n, dtype=torch.float64)[:, None] * theta ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    return at.cos().float().cuda(), at.sin().float().cuda()


def rotated(x, cos, sin):
    """fp32 x [n, heads, hd] with the rotation of each row, products and sums rounded one by one; and the same in 64 bits."""
    e, o = x[..., 0::2], x[..., 1::2]
    c, s = cos[:, None], sin[:, None]
    f = torch.stack([e * c - o * s, o * c + e * s], -1).flatten(-2)
    e, o, c, s = e.double(), o.double(), c.double(), s.double()
    return f, torch.stack([e * c - o * s, o * c + e * s], -1).flatten(-2)


def power_of_two(largest):
    """The smallest power of two, at least 2^-126, that brings `largest` (numpy fp32) within 448."""
    out = np.empty_like(largest)
    for i, x in np.ndenumerate(largest):
        m, e = math.frexp(float(x) / 448.0)
        out[i] = 2.0 ** max((e - 1 if m == 0.5 else e) if x > 0 else -126, -126)
    return out


def attention_exact(q, k, v, pos, scale, window):
    """q [n, heads, hd], k and v [len, kv, hd] in 64 bits; what the rows at positions pos.. see.  Also sum of p |v| and the largest
    sum of |q| |k| of a row, for tolerances."""
    n, h, hd = q.shape
    g = h // k.shape[1]
    k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    s = torch.einsum("nhd,lhd->hnl", q, k) * scale
    at = torch.arange(k.shape[0])
    mine = (pos + torch.arange(n))[:, None]
    hidden = at > mine
    if window:
        hidden |= at <= mine - window
    s = s.masked_fill(hidden, -math.inf)
    p = torch.softmax(s, -1)
    big = (torch.einsum("nhd,lhd->hnl", q.abs(), k.abs()) * scale).masked_fill(hidden, 0).amax(-1)
    return torch.einsum("hnl,lhd->nhd", p, v), torch.einsum("hnl,lhd->nhd", p, v.abs()), big.T


def attention_tolerance(ref, mass, big, kind, hd, length, q, scale, kmax):
    """How far a bf16 result may be off.  Scores: sums of hd products on the tensor cores, 2^-23 of the sum of magnitudes a step of 16 and
    some more for scaling, exponent and (8-bit caches) the queries' conversion.  Probabilities: rounded to bf16 (2^-8) or f16 (2^-11).
    Sums over keys: 2^-23 a step of 16, and as much for the statistics.  The result: rounded to bf16."""
    ds = (hd / 16 + 8) * 2.0 ** -22 * big + 2.0 ** -20 + hd * 2.0 ** -33 * float(q.abs().max()) * kmax * scale
    dp = (2.0 ** -8 if kind == "bf16" else 2.0 ** -11) + 2 * ds + (length / 16 + 64) * 2.0 ** -22
    return 2.0 ** -8 * ref.abs() + dp[..., None] * mass * (1 + 2.0 ** -7) + 1e-30


def rules_args(logits, out, **kw):
    a = _ffi.LogitRulesArgs(struct_size=ctypes.sizeof(_ffi.LogitRulesArgs),
                            dtype=_ffi.DTYPE_F32 if logits.dtype == torch.float32 else _ffi.DTYPE_BF16, d_logits=ptr(logits),
                            d_out=ptr(out), ld_logits=logits.stride(0), ld_out=out.stride(0), rows=logits.shape[0],
                            vocab=logits.shape[1])
    for k, v in kw.items():
        setattr(a, k, ptr(v) if isinstance(v, torch.Tensor) else v)
    a.keep = kw
    return a


def rules(logits, out, **kw):
    a = rules_args(logits, out, **kw)
    rc = lib.ane_op_logit_rules(ctypes.byref(a))
    assert rc == 0, lib.ane_ops_last_error()
