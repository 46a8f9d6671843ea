"""GPU: windows, forks, packing and beam search through the engine, together."""
import numpy as np
import pytest
import torch

from oracle.model_ref import synth_weights_numpy

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def weights():
    from higgs_b200.model import tiny_args, weights_to_device
    out = {}
    for kind in ("qwen3", "llama"):
        args = tiny_args(kind, 2)
        out[kind] = args, weights_to_device(synth_weights_numpy(args, seed=0), DEV)
    return out


def engine(weights, kind="qwen3", pages=128, max_seq_len=256, kv_mode="bf16", **kw):
    from higgs_b200.engine import Engine
    from higgs_b200.model import Model
    args, w = weights[kind]
    return Engine(Model(args, w, num_pages=pages, device=DEV, kv_mode=kv_mode, **kw), max_seq_len=max_seq_len,
                  keep_logits=True)


# Logits of two passes over the same tokens (a prompt against decode steps: other kernels, other
# orders of sums).  Each is within atol 2e-2 + rtol 1e-2 of the model computed exactly (the bar of
# test_model_gpu.py), so by the triangle inequality the two are within twice that of each other.
TWO_PASSES = dict(atol=2 * 2e-2, rtol=2 * 1e-2)


def prompt(n, seed=1, vocab=4096):
    return np.random.default_rng(seed).integers(0, vocab, n).astype(np.int32)


def steps(eng, seqs, n):
    """(tokens, logits of every step)"""
    eng.step_logits.clear()
    t = eng.decode_steps(seqs, n)
    return t, np.stack(eng.step_logits)


@pytest.mark.parametrize("kind", ["qwen3", "llama"])
def test_window_as_long_as_the_cache_is_the_plain_model(weights, kind):
    """The same logits for a 70-token prompt and 12 decode steps, by other attention kernels."""
    a, b = engine(weights, kind), engine(weights, kind, attn_window=256)
    sa, sb = a.prefill(prompt(70), use_prefix=False), b.prefill(prompt(70), use_prefix=False)
    np.testing.assert_allclose(sa.first_logits, sb.first_logits, **TWO_PASSES)
    force = prompt(12, seed=3)[None]
    a.decode_steps([sa], 12, force=force)
    b.decode_steps([sb], 12, force=force)
    np.testing.assert_allclose(np.stack(a.step_logits), np.stack(b.step_logits), **TWO_PASSES)


@pytest.mark.parametrize("window,sinks", [(24, 4), (40, 0), (17, 20)])
def test_window_decode_gives_up_pages(weights, window, sinks):
    """A windowed model: decode steps agree with one prompt pass over the same tokens (the other
    attention kernel), pages behind the window return to the pool, and what is then written into
    them changes nothing."""
    eng = engine(weights, attn_window=window, attn_sinks=sinks)
    pr, force = prompt(90), prompt(60, seed=5)[None]
    seq = eng.prefill(pr, use_prefix=False)
    free0 = eng.pool.num_free
    eng.step_logits.clear()
    eng.decode_steps([seq], 30, force=force[:, :30])
    live = [p for p in seq.pages if p >= 0]
    need = -(-sinks // 16) + -(-window // 16) + 2
    assert len(live) <= need and len(seq.pages) == 8 and eng.pool.num_free > free0 - 2
    # the pages that were given up are other sequences' now
    other = eng.prefill(prompt(100, seed=9), use_prefix=False)
    eng.decode_steps([seq], 30, force=force[:, 30:])
    got = np.stack(eng.step_logits)[:, 0]
    eng.release(other)
    eng.release(seq)
    whole = np.concatenate([pr, force[0]])
    ref = engine(weights, attn_window=window, attn_sinks=sinks)
    for k in (0, 13, 29, 30, 59):
        want = ref.prefill(whole[:91 + k], use_prefix=False).first_logits
        np.testing.assert_allclose(got[k], want, **TWO_PASSES)
    assert eng.pool.num_free == 128


@pytest.mark.parametrize("kv_mode,length", [("bf16", 37), ("bf16", 48), ("tq4", 37)])
def test_fork_continues_alike_and_apart(weights, kv_mode, length):
    eng = engine(weights, kv_mode=kv_mode)
    seq = eng.prefill(prompt(length), use_prefix=False)
    twin, third = eng.fork(seq, 2)
    assert twin.pages[:length // 16] == seq.pages[:length // 16]
    t, lg = steps(eng, [seq, twin, third], 20)
    assert np.array_equal(t[0], t[1]) and np.array_equal(lg[:, 0], lg[:, 1]) and np.array_equal(lg[:, 0], lg[:, 2])
    # each goes its own way without touching the others'
    alone = engine(weights, kv_mode=kv_mode)
    ref = alone.prefill(prompt(length), use_prefix=False)
    alone.decode_steps([ref], 20)
    force = np.stack([prompt(10, seed=s) for s in (1, 2, 3)])
    eng.step_logits.clear()
    eng.decode_steps([seq, twin, third], 10, force=force)
    copy = eng.fork(third)[0]
    assert len(set(copy.pages) & set(third.pages)) == (length + 30) // 16
    for s in (seq, twin, third, copy):
        eng.release(s)
    assert eng.pool.num_free == 128


@pytest.mark.parametrize("kv_mode", ["bf16", "tq4"])
def test_compact_keeps_generations(weights, kv_mode):
    """Packing the pool between steps changes page ids and nothing else: bit-equal logits, prefix
    hits included."""
    runs = []
    for pack in (False, True):
        eng = engine(weights, kv_mode=kv_mode)
        hole = eng.prefill(prompt(100, seed=7), use_prefix=False)
        a = eng.prefill(prompt(50, seed=1))
        hole2 = eng.prefill(prompt(60, seed=8), use_prefix=False)
        b = eng.prefill(prompt(33, seed=2), use_prefix=False)
        steps(eng, [a, b], 5)
        eng.release(hole)
        eng.release(hole2)
        if pack:
            moved = eng.compact([a, b])
            assert moved > 0 and max(a.pages + b.pages) < eng.pool.num_pages - eng.pool.num_free
        t, lg = steps(eng, [a, b], 20)
        c = eng.prefill(np.concatenate([prompt(50, seed=1), prompt(5, seed=4)]))
        assert c.prefix_hit == 48
        runs.append((t, lg, c.first_logits))
    for x, y in zip(*runs):
        assert np.array_equal(x, y)


def log_softmax(x):
    x = x.astype(np.float64)
    return x - x.max() - np.log(np.exp(x - x.max()).sum())


def test_beam_of_one_is_greedy(weights):
    eng = engine(weights)
    want = eng.generate_greedy([prompt(40)], 12, use_prefix=False)[0]
    toks, scores = eng.generate_beam(prompt(40), 1, 12, use_prefix=False)
    assert np.array_equal(toks[0], want) and eng.pool.num_free == 128


@pytest.mark.parametrize("kw", [{}, {"attn_window": 24, "attn_sinks": 4}, {"kv_mode": "tq4"}])
def test_beam_search_scores(weights, kw):
    """Scores are the log-probabilities of their tokens in a pass over the whole sequence, best
    first; no hypothesis twice; every page is back afterwards; the best is no worse than the
    greedy one."""
    eng = engine(weights, **kw)
    pr, n = prompt(45, seed=6), 9
    toks, scores = eng.generate_beam(pr, 4, n, use_prefix=False)
    assert len(toks) == 4 and all(t.size == n for t in toks) and len({t.tobytes() for t in toks}) == 4
    assert (np.diff(scores) <= 0).all() and eng.pool.num_free == 128
    greedy = eng.generate_greedy([pr], n, use_prefix=False)[0]
    ref = engine(weights, **kw)

    def rescore(t):
        s = 0.0
        for i in range(n):
            q = ref.prefill(np.concatenate([pr, t[:i]]), use_prefix=False)
            s += log_softmax(q.first_logits)[t[i]]
            ref.release(q)
        return s / n
    # a step's logits of two passes are within twice 2e-2 + 1e-2 |x| (above), |x| < 3 here, and a log
    # sum moves by no more than its largest logit: the difference of the two by at most twice that
    tol = 2 * 2 * (2e-2 + 1e-2 * 3)
    for t, s in zip(toks, scores):
        assert abs(rescore(t) - s) < tol
    assert scores[0] >= rescore(greedy) - tol


def test_beam_search_ends_at_eos(weights):
    eng = engine(weights)
    pr = prompt(20, seed=2)
    plain, _ = eng.generate_beam(pr, 3, 8, use_prefix=False)
    eos = int(plain[0][3])
    toks, scores = eng.generate_beam(pr, 3, 8, eos_token_id=eos, use_prefix=False)
    assert len(toks) == 3 and (np.diff(scores) <= 0).all() and eng.pool.num_free == 128
    for t in toks:
        hits = np.nonzero(t == eos)[0]
        assert t.size == 8 or (hits.size == 1 and hits[0] == t.size - 1)


def test_beam_search_prefers_longer_with_penalty(weights):
    eng = engine(weights)
    a = eng.generate_beam(prompt(30), 4, 6, length_penalty=0.0, use_prefix=False)
    b = eng.generate_beam(prompt(30), 4, 6, length_penalty=1.0, use_prefix=False)
    assert all(np.array_equal(x, y) for x, y in zip(a[0], b[0]))
    np.testing.assert_allclose(a[1], b[1] * 6, rtol=1e-12)


def test_beam_search_refuses(weights):
    eng = engine(weights)
    for kw in (dict(beams=0), dict(beams=17), dict(max_new_tokens=0), dict(max_new_tokens=300)):
        with pytest.raises(ValueError):
            eng.generate_beam(prompt(20), **{"beams": 2, "max_new_tokens": 4, **kw})
    assert eng.pool.num_free == 128
    small = engine(weights, pages=4)
    from higgs_b200.ffi import HiggsError
    with pytest.raises(HiggsError):
        small.generate_beam(prompt(40), 4, 8, use_prefix=False)  # no page left for the forks
    assert small.pool.num_free == 4


def test_windowed_model_refuses_tq4(weights):
    from higgs_b200.ffi import HiggsError
    with pytest.raises(HiggsError, match="TurboQuant"):
        engine(weights, kv_mode="tq4", attn_window=16)


@pytest.mark.parametrize("kv_mode,kw", [("bf16", {}), ("bf16", {"attn_window": 24}), ("tq4", {})])
def test_speculative_decoder_made_late_leaves_the_cache(weights, kv_mode, kw):
    """Making a SpecDecoder (its warm-up and capture) writes nothing into pages that sequences own."""
    from higgs_b200.engine import SpecDecoder
    eng = engine(weights, kv_mode=kv_mode, **kw)
    seq = eng.prefill(prompt(40), use_prefix=False)
    torch.cuda.synchronize()
    before = [p.clone() for p in eng.model.kv_pools]
    dec = SpecDecoder(eng, 2, k=3, draft_layers=1, temperature=0.0)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, eng.model.kv_pools))
    dec.stage([seq, eng.fork(seq)[0]], np.zeros(2 * 3 * 2 + 2, np.float32), first=True)
    dec.graph.replay()
    torch.cuda.synchronize()
    assert not all(torch.equal(a, b) for a, b in zip(before, eng.model.kv_pools))


def test_window_speculative_steps_give_up_pages(weights):
    """Speculative steps of a windowed model: the same tokens whether the pages behind the window go
    back to the pool (where another sequence takes and fills them) or stay."""
    from higgs_b200.engine import SpecDecoder
    runs = []
    for trim in (True, False):
        eng = engine(weights, attn_window=24, attn_sinks=4)
        if not trim:
            eng._trim = lambda s: None
        seqs = [eng.prefill(prompt(n, seed=n), use_prefix=False) for n in (90, 40)]
        dec = SpecDecoder(eng, 2, k=3, draft_layers=1, temperature=0.0)
        rng = np.random.default_rng(0)
        dec.steps(seqs, 8, rng)
        other = eng.prefill(prompt(100, seed=9), use_prefix=False)  # fills the pages that were given up
        acc = dec.steps(seqs, 8, rng)
        live = [sum(p >= 0 for p in s.pages) for s in seqs]
        if trim:  # sinks, window and the tokens ahead
            assert max(live) <= 1 + 4 and all(s.pages[2] == -1 for s in seqs[:1])
        runs.append(([list(s.generated) for s in seqs], acc))
        for s in seqs + [other]:
            eng.release(s)
        assert eng.pool.num_free == 128
    assert runs[0][0] == runs[1][0] and np.array_equal(runs[0][1], runs[1][1])


@pytest.mark.parametrize("kv_mode,length", [("bf16", 37), ("bf16", 48), ("tq4", 37)])
def test_forks_that_go_apart_are_sequences_of_their_own(weights, kv_mode, length):
    """Three forks fed different tokens give, bit for bit, the logits of three sequences that never
    shared a page (the same batch, so the same kernels)."""
    force = np.stack([prompt(40, seed=s) for s in (1, 2, 3)])
    runs = []
    for forked in (True, False):
        eng = engine(weights, kv_mode=kv_mode)
        if forked:
            first = eng.prefill(prompt(length), use_prefix=False)
            seqs = [first] + eng.fork(first, 2)
        else:
            seqs = [eng.prefill(prompt(length), use_prefix=False) for _ in range(3)]
        eng.step_logits.clear()
        eng.decode_steps(seqs, 20, force=force[:, :20])
        if forked:  # the first one's place is taken by a fork of it, made in the middle
            seqs = eng.fork(seqs[0]) + seqs[1:]
            eng.release(first)
        eng.decode_steps(seqs, 20, force=force[:, 20:])
        runs.append(np.stack(eng.step_logits))
        for s in seqs:
            eng.release(s)
        assert eng.pool.num_free == 128
    assert np.array_equal(runs[0], runs[1])
    assert not np.array_equal(runs[0][-1, 0], runs[0][-1, 1])
