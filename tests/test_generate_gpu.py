"""Engine.generate: prompts of different lengths over paged caches of bf16 or 8 bits, with rules on the logits, against the engine's own
full forward pass on the tokens that came out."""
import numpy as np
import pytest

import ane
from oracle import oracle as O
from parity_utils import make_pair

pytestmark = pytest.mark.gpu
CLEAR = 0.05  # between the two best logits: what bf16 noise cannot turn round (the margin of the dense cache's tests)


def pair(batch=4, std=0.08, **over):
    cfg = dict(dim=256, hidden=512, heads=4, kv_heads=2, layers=3, vocab=2048, seq=160)
    cfg.update(over)
    m, e = make_pair(ane, dict(cfg), arch=O.ARCH_L, quirks=0, dtype=ane.DTYPE_BF16, batch=batch, std=std, debug_taps=False)
    cfg["exact"] = m
    return cfg, e


def forward(e, cfg, prompt, out):
    """Logits [vocab] of each position that chose a token, from a forward pass over the whole sequence."""
    full = np.zeros(cfg["seq"], dtype=np.uint16)
    full[:len(prompt)] = prompt
    full[len(prompt):len(prompt) + len(out)] = out
    logits = e.eval_logits(full)[0]
    return [logits[:, len(prompt) - 1 + i] for i in range(len(out))]


def ruled(x, prompt, said, repetition, presence, frequency, bias, allowed):
    x = x.astype(np.float32).copy()
    for t in set(prompt) | set(said):
        x[t] = x[t] / np.float32(repetition) if x[t] > 0 else x[t] * np.float32(repetition)
    for t in set(said):
        x[t] -= np.float32(frequency) * np.float32(said.count(t)) + np.float32(presence)
    for t, b in bias.items():
        x[t] += np.float32(b)
    if allowed is not None:
        x[~allowed] = -np.inf
    return x


@pytest.mark.parametrize("heads", [(4, 2), (4, 4), (8, 1)])
def test_generate_bf16_matches_own_full_forward(heads):
    cfg, e = pair(heads=heads[0], kv_heads=heads[1])  # head sizes 64 and 32
    toks = O.zipf_tokens(300, cfg["vocab"], 9)
    prompts = [toks[:64], toks[64:65], toks[70:200], toks[200:233]]
    got = e.generate(prompts, 24)
    agree = total = 0
    for b, p in enumerate(prompts):
        for i, col in enumerate(forward(e, cfg, p, got[b])):
            top2 = np.sort(col)[-2:]
            if top2[1] - top2[0] > CLEAR:
                total += 1
                agree += int(col.argmax() == got[b, i])
    assert total > 20 and agree == total
    e.close()


def test_generate_gives_what_the_dense_cache_gives():
    cfg, e = pair()
    prompts = O.zipf_tokens(4 * 50, cfg["vocab"], 4).reshape(4, 50)
    a, b = e.generate(list(prompts), 30), e.decode_greedy(prompts, 30)
    for s in range(4):
        cols = forward(e, cfg, prompts[s], b[s])
        for i in range(30):
            if a[s, i] != b[s, i]:  # only where two tokens are as good as each other
                top2 = np.sort(cols[i])[-2:]
                assert top2[1] - top2[0] <= CLEAR
                break
    assert np.array_equal(a, e.generate(list(prompts), 30))  # the same again, with used pages
    e.close()


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
def test_generate_with_rules_matches_own_full_forward(kv):
    cfg, e = pair(std=0.1)
    rng = np.random.default_rng(3)
    toks = O.zipf_tokens(200, cfg["vocab"], 5)
    prompts = [toks[:40], toks[40:47], toks[50:150]]
    allowed = rng.random(cfg["vocab"]) < 0.5
    bias = {int(t): float(b) for t, b in zip(rng.integers(0, cfg["vocab"], 20), rng.standard_normal(20))}
    rules = dict(repetition=1.3, presence=0.4, frequency=0.2)
    got = e.generate(prompts, 30, kv=kv, bias=bias, allowed=allowed, **rules)
    assert allowed[got].all()
    for b, p in enumerate(prompts):
        cols = forward(e, cfg, p, got[b])
        full = np.zeros(cfg["seq"], dtype=np.uint16)
        full[:len(p) + 30] = np.concatenate([p, got[b]])
        exact = cfg["exact"].eval_logits(full)[:, len(p) - 1:len(p) + 29]  # fp32
        # The choice is the best by logits that are off by about as much as those here, which are off by `off` from fp32 ones: two logits in
        # two passes, and the repetition penalty stretches what is negative.
        off = float(np.abs(np.stack(cols, 1) - exact).max())
        for i, col in enumerate(cols):
            x = ruled(col, [int(t) for t in p], [int(t) for t in got[b, :i]], bias=bias, allowed=allowed, **rules)
            # 8 bits: keys and values off by up to 2^-4 each; what is asked is that the choice is among the best, by the spread of logits
            margin = 4 * 1.3 * off if kv == "bf16" else 0.5 * float(col.std())
            assert x.max() - x[got[b, i]] <= margin, (b, i, x.max() - x[got[b, i]], off)
    e.close()


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
def test_generate_follows_a_sure_model(kv):
    """Weights that know their next token (the classifier finds the code that the first feed-forward block moved): the chain comes out whatever
    type the cache has."""
    cfg, e = pair(heads=4, kv_heads=2, vocab=512, batch=3, std=0.002)
    rng = np.random.default_rng(1)
    dim, hidden, vocab, half = cfg["dim"], cfg["hidden"], cfg["vocab"], cfg["dim"] // 2
    code = rng.standard_normal((vocab, half)).astype(np.float32)
    follows = rng.permutation(vocab)
    e.import_tensor(ane.T_EMBED, 0, 0.1 * np.concatenate([code, code[follows]], 1))
    w1, w2 = np.zeros((hidden, dim), np.float32), np.zeros((dim, hidden), np.float32)
    at = np.arange(half)
    w1[at, half + at], w1[half + at, half + at] = 1, -1
    w2[at, at], w2[at, half + at] = 1, -1
    e.import_tensor(ane.T_W1, 0, w1)
    e.import_tensor(ane.T_W3, 0, w1)
    e.import_tensor(ane.T_W2, 0, w2)
    prompts = [[3], [7, 8, 9] * 20, list(range(33))]
    got = e.generate(prompts, 60, kv=kv)
    for p, g in zip(prompts, got):
        t = p[-1]
        for x in g:
            t = follows[t]
            assert x == t
    # one token biased above all, and the token that would follow forbidden
    assert (e.generate(prompts, 5, kv=kv, bias={17: 1e4}) == 17).all()
    allowed = np.ones(vocab, bool)
    allowed[follows[3]] = False
    g = e.generate([[3]], 1, kv=kv, allowed=allowed)
    assert g[0, 0] != follows[3]
    # sampling: draws decide, and the same draws give the same tokens; a sure model follows its chain at a low temperature
    u = rng.random((60, 3))
    cold = e.generate(prompts, 60, kv=kv, temperature=0.01, uniforms=u)
    assert np.array_equal(cold, got)
    hot = e.generate(prompts, 60, kv=kv, temperature=50.0, uniforms=u)
    assert np.array_equal(hot, e.generate(prompts, 60, kv=kv, temperature=50.0, uniforms=u)) and not np.array_equal(hot, got)
    e.close()


def test_generate_fills_the_window_and_more_sequences_than_the_dense_kernels_take():
    cfg, e = pair(batch=40, seq=100, layers=2)
    prompts = [O.zipf_tokens(1 + 2 * b, cfg["vocab"], b) for b in range(40)]
    got = e.generate(prompts, 100 - 79, kv="e4m3")
    assert got.shape == (40, 21)
    got = e.generate(prompts[:1], 99)  # the window's last place
    cols = forward(e, cfg, prompts[0], got[0])
    for i, col in enumerate(cols):
        assert col.max() - col[got[0, i]] <= CLEAR
    e.close()


def test_generate_refuses():
    cfg, e = pair(batch=2)
    ok = [[1, 2, 3]]
    for kw in (dict(prompts=[], n_new=1), dict(prompts=ok * 3, n_new=1), dict(prompts=[[]], n_new=1), dict(prompts=ok, n_new=0),
               dict(prompts=ok, n_new=158), dict(prompts=ok, n_new=161), dict(prompts=ok, n_new=1, temperature=1.0), dict(prompts=ok, n_new=1, kv="int8"),
               dict(prompts=ok, n_new=1, repetition=-1.0), dict(prompts=ok, n_new=1, repetition=float("nan")),
               dict(prompts=ok, n_new=1, presence=float("nan")), dict(prompts=ok, n_new=1, allowed=np.zeros(cfg["vocab"], bool)),
               dict(prompts=ok, n_new=1, allowed=np.ones(3, bool)), dict(prompts=ok, n_new=1, bias={i: 1.0 for i in range(1025)}),
               dict(prompts=ok, n_new=2, temperature=1.0, uniforms=np.zeros((1, 1)))):
        with pytest.raises(ane.EngineError):
            e.generate(**kw)
    assert e.generate(ok, 157).shape == (1, 157)
    e.close()
    with pytest.raises(ane.EngineError):
        e.generate(ok, 1)
    small = dict(dim=64, hidden=96, heads=4, layers=2, vocab=256, seq=32)
    for arch, dtype in ((O.ARCH_N, ane.DTYPE_BF16), (O.ARCH_L, ane.DTYPE_F32), (O.ARCH_L, ane.DTYPE_BF16)):  # the last: head size 16
        _, e = make_pair(ane, small, arch=arch, quirks=0, dtype=dtype, batch=1, debug_taps=False)
        with pytest.raises(ane.EngineError):
            e.generate(ok, 1)
        e.close()


def test_generate_leaves_training_as_it_was():
    cfg, e = pair(batch=2)
    toks = O.zipf_tokens(2 * 161, cfg["vocab"], 7).reshape(2, 161)
    inp, tgt = np.ascontiguousarray(toks[:, :160]), np.ascontiguousarray(toks[:, 1:])
    before = e.step_tokens(inp, tgt).loss
    cfg, f = pair(batch=2)
    f.generate([toks[0, :50], toks[1, :9]], 20, kv="e4m3")
    f.decode_greedy(toks[:, :20], 10)
    assert f.step_tokens(inp, tgt).loss == before
    e.close()
    f.close()
