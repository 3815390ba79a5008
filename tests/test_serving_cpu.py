"""Refusals of the serving operators: arguments are checked before anything touches a device."""
import ctypes

import pytest
from ane import _ffi

lib = _ffi.lib
HERE = 1 << 20  # stands for a device address; refused calls do not use it


def cache(**over):
    c = _ffi.KvCache(struct_size=ctypes.sizeof(_ffi.KvCache), dtype=_ffi.KV_E4M3, d_k=HERE, d_v=HERE, d_k_scale=HERE, d_v_scale=HERE,
                     n_pages=4, page_size=16, n_kv_heads=2, head_dim=64, d_page_table=HERE, table_pitch=2)
    for k, v in over.items():
        setattr(c, k, v)
    return c


def append(c=None, **over):
    a = _ffi.KvAppendArgs(struct_size=ctypes.sizeof(_ffi.KvAppendArgs), n_heads=4, cache=ctypes.pointer(c or cache()), d_qkv=HERE, d_q=HERE + 4096,
                          ld_qkv=8 * 64, ld_q=4 * 64, d_cos=HERE, d_sin=HERE, n_positions=10, n_seq=1, d_seq_start=HERE, d_pos=HERE, n_tokens=1)
    for k, v in over.items():
        setattr(a, k, v)
    return lib.ane_op_kv_append(ctypes.byref(a))


def attention(c=None, **over):
    a = _ffi.KvAttentionArgs(struct_size=ctypes.sizeof(_ffi.KvAttentionArgs), n_heads=4, cache=ctypes.pointer(c or cache()), d_q=HERE, d_out=HERE,
                             ld_q=4 * 64, ld_out=4 * 64, d_seq_start=HERE, d_pos=HERE, n_seq=1, n_tokens=1, max_new=1, d_workspace=HERE)
    for k, v in over.items():
        setattr(a, k, v)
    return lib.ane_op_kv_attention(ctypes.byref(a))


def rules(**over):
    a = _ffi.LogitRulesArgs(struct_size=ctypes.sizeof(_ffi.LogitRulesArgs), dtype=_ffi.DTYPE_F32, d_logits=HERE, d_out=HERE, ld_logits=100,
                            ld_out=100, rows=2, vocab=100)
    for k, v in over.items():
        setattr(a, k, v)
    return lib.ane_op_logit_rules(ctypes.byref(a))


def refused(rc, word):
    assert rc == -1
    assert word.encode() in lib.ane_ops_last_error(), lib.ane_ops_last_error()


CACHES = [
    (dict(struct_size=8), "struct_size"), (dict(dtype=2), "dtype"), (dict(head_dim=80), "head_dim"), (dict(page_size=0), "page_size"),
    (dict(page_size=24), "page_size"), (dict(page_size=8192), "page_size"), (dict(n_pages=0), "dimensions"), (dict(n_kv_heads=0), "dimensions"),
    (dict(n_kv_heads=3), "n_heads"), (dict(table_pitch=0), "dimensions"), (dict(d_k=None), "null"), (dict(d_v=None), "null"),
    (dict(d_k_scale=None), "null"), (dict(d_v_scale=None), "null"), (dict(d_page_table=None), "null"), (dict(d_k=HERE + 8), "aligned"),
    (dict(d_v=HERE + 1), "aligned"), (dict(page_stride=2047), "page_stride"), (dict(page_stride=2056), "page_stride"),
    (dict(page_stride=-2048), "page_stride"), (dict(page_stride=1 << 40), "64 GiB"), (dict(page_stride=1 << 62, n_pages=2 ** 31 - 1), "64 GiB"),
]


@pytest.mark.parametrize("over,word", CACHES)
def test_caches_that_make_no_sense_are_refused(over, word):
    refused(append(cache(**over)), word)
    refused(attention(cache(**over)), word)


@pytest.mark.parametrize("over,word", [
    (dict(struct_size=0), "struct_size"), (dict(n_heads=0), "n_heads"), (dict(n_heads=3), "n_heads"), (dict(d_qkv=None), "null"),
    (dict(d_seq_start=None), "null"), (dict(d_pos=None), "null"), (dict(n_seq=-1), "number"), (dict(n_tokens=-1), "number"),
    (dict(d_qkv=HERE + 2), "aligned"), (dict(d_q=HERE + 2), "aligned"), (dict(ld_qkv=8 * 64 - 8), "ld_qkv"), (dict(ld_qkv=8 * 64 + 4), "ld_qkv"),
    (dict(ld_q=4 * 64 - 8), "ld_q"), (dict(ld_q=4 * 64 + 1), "ld_q"), (dict(d_q=HERE), "in place"), (dict(d_cos=None), "missing"),
    (dict(d_sin=None), "missing"), (dict(n_positions=0), "positions"), (dict(d_cos=HERE + 4), "aligned"),
])
def test_append_refuses(over, word):
    refused(append(**over), word)


@pytest.mark.parametrize("over,word", [
    (dict(struct_size=0), "struct_size"), (dict(d_q=None), "null"), (dict(d_out=None), "null"), (dict(d_workspace=None), "null"),
    (dict(d_q=HERE + 2), "aligned"), (dict(d_out=HERE + 8), "aligned"), (dict(d_workspace=HERE + 8), "aligned"), (dict(ld_q=248), "ld_q"),
    (dict(ld_out=260), "ld_out"), (dict(max_new=0), "max_new"), (dict(max_new=2 ** 30), "max_new"), (dict(window=-1), "window"),
    (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(n_seq=-1), "number"),
])
def test_attention_refuses(over, word):
    refused(attention(**over), word)


def test_attention_workspace_refuses():
    for bad in ((0, 1, 64), (4, 0, 64), (4, 3, 64), (4, 2, 65)):
        assert lib.ane_op_kv_attention_workspace(*bad) == 0
        assert b"bad heads" in lib.ane_ops_last_error()


@pytest.mark.parametrize("over,word", [
    (dict(struct_size=0), "struct_size"), (dict(dtype=2), "fp32 or bf16"), (dict(d_logits=None), "null"), (dict(d_out=None), "null"),
    (dict(rows=-1), "dimensions"), (dict(vocab=0), "dimensions"), (dict(ld_logits=99), "dimensions"), (dict(ld_out=99), "dimensions"),
    (dict(d_logits=HERE + 2), "misaligned"), (dict(d_out=HERE + 1), "misaligned"), (dict(dtype=_ffi.DTYPE_BF16), "in place"),
    (dict(ld_out=104), "in place"), (dict(d_tokens=HERE, ld_tokens=4), "token"), (dict(d_tokens=HERE, d_n_tokens=HERE), "token"),
    (dict(d_tokens=HERE, d_n_tokens=HERE, ld_tokens=1 << 24), "token"), (dict(d_repetition=HERE), "penalties"), (dict(d_presence=HERE), "penalties"),
    (dict(d_frequency=HERE), "penalties"), (dict(d_mask=HERE, ld_mask=3, n_masks=2), "masks"), (dict(d_mask=HERE, ld_mask=4, n_masks=1), "masks"),
    (dict(d_mask=HERE, d_mask_row=HERE, ld_mask=4, n_masks=0), "masks"), (dict(d_bias_start=HERE), "biases"),
    (dict(d_bias_start=HERE, d_bias=HERE), "biases"), (dict(d_bias_start=HERE, d_bias_token=HERE), "biases"),
])
def test_rules_refuse(over, word):
    refused(rules(**over), word)


def test_null_arguments_are_refused():
    assert lib.ane_op_kv_append(None) == -1
    assert lib.ane_op_kv_attention(None) == -1
    assert lib.ane_op_logit_rules(None) == -1
