"""CPU: Engine.generate_beam against a plain beam search, with a stand-in for the device: logits are a
function of the tokens found in the sequence's own pages, so a wrong fork, copy or page shows."""
import math

import numpy as np
import pytest
import torch

from higgs_b200.engine import PAGE, Engine, Sequence
from higgs_b200.kv import BlockPool, PrefixCache
from higgs_b200 import ops


class _Model:
    device, tp, attn_window, attn_sinks = "cpu", None, 0, 0

    def __init__(self, vocab):
        class Args:
            vocab_size = vocab
        self.args = Args


class _Graph:
    def __init__(self, eng):
        self.eng = eng

    def run(self):
        self.logits = torch.from_numpy(np.stack([self.eng.logits_of(s) for s in self.eng.staged]))


class StandIn(Engine):
    """The engine over a cache that holds one token id per slot."""

    def __init__(self, vocab, pages, logits, max_seq_len):
        self.model = _Model(vocab)
        self.pool = BlockPool(pages)
        self.prefix = PrefixCache(self.pool, 4)
        self.max_seq_len = max_seq_len
        self.keep_logits = False
        self.cache = np.full((pages, PAGE), -1, np.int64)
        self.logits = logits

    def logits_of(self, s):
        toks = [int(self.cache[s.pages[i // PAGE], i % PAGE]) for i in range(s.length)]
        return self.logits(tuple(toks))

    def _append(self, s, token):
        self._ensure_pages(s, s.length + 1)
        self.cache[s.pages[s.length // PAGE], s.length % PAGE] = token
        s.length += 1

    def _prefill(self, prompt, use_prefix, want_logits):
        s = Sequence(prompt=np.asarray(prompt, np.int32))
        for t in prompt:
            self._append(s, t)
        return s, torch.from_numpy(self.logits_of(s)[None])

    def _graph_for_logits(self, B):
        return _Graph(self)

    def stage_step(self, seqs, g, first):
        assert len({p for s in seqs for p in s.pages[s.length // PAGE:]}) == \
            sum(len(s.pages) - s.length // PAGE for s in seqs), "two sequences would write one page"
        for s in seqs:
            self._append(s, s.last_token)
        self.staged = seqs

    def _copy_pages(self, src, dst):
        for a, b in zip(src, dst):
            self.cache[b] = self.cache[a]


def _select(logits, scores, n_out, workspace=None):
    """higgs_beam_select as it is defined: keys in 64 bits, rounded to f32."""
    B, W = scores.shape
    key = scores.double()[:, :, None] + torch.log_softmax(logits.double().view(B, W, -1), 2)
    flat = key.view(B, -1)
    order = torch.from_numpy(np.argsort(-flat.numpy(), 1, kind="stable")[:, :n_out].copy())
    best = flat.gather(1, order)
    V = key.shape[2]
    none = torch.isinf(best)
    return (best.float(), torch.where(none, -1, order // V).int(), torch.where(none, -1, order % V).int())


@pytest.fixture(autouse=True)
def selection(monkeypatch):
    monkeypatch.setattr(ops, "beam_select", _select)
    monkeypatch.setattr(ops, "beam_select_workspace", lambda *a: None)


def hashed_logits(vocab, sd=2.0):
    def f(toks):
        seed = 0
        for t in toks:
            seed = (seed * 1000003 + t + 12345) % (2 ** 63)
        return np.random.default_rng(seed).normal(0, sd, vocab).astype(np.float32)
    return f


def plain_search(logits, prompt, beams, steps, eos, penalty):
    """The search as generate_beam documents it, over recomputed logits in 64 bits."""
    live, done = [(0.0, ())], []
    for step in range(1, steps + 1):
        cand = []
        for w, (total, toks) in enumerate(live):
            x = logits(tuple(prompt) + toks).astype(np.float64)
            lp = x - x.max() - math.log(np.exp(x - x.max()).sum())
            cand += [(-(total + lp[v]), w, v) for v in range(len(x))]
        live, ahead = [], live
        for s, w, v in sorted(cand)[:2 * beams]:
            if len(live) == beams:
                break
            if v == eos:
                done.append((-s / step ** penalty, ahead[w][1] + (v,)))
            else:
                live.append((-s, ahead[w][1] + (v,)))
        done = sorted(done, key=lambda d: -d[0])[:beams]
        if not live:
            break
        best_ahead = max(live[0][0] / k ** penalty for k in (step, steps))
        if step == steps or (len(done) == beams and best_ahead <= done[-1][0]):
            done = sorted(done + [(s / step ** penalty, t) for s, t in live], key=lambda d: -d[0])[:beams]
            break
    return [t for _, t in done], [s for s, _ in done]


@pytest.mark.parametrize("beams,steps,eos,penalty,n", [(1, 10, None, 1.0, 5), (4, 40, None, 1.0, 30), (4, 40, 3, 1.0, 16),
                                                       (3, 25, 3, 0.0, 17), (5, 25, 3, 2.0, 31), (16, 20, 7, 1.0, 1),
                                                       (2, 1, 3, 1.0, 15), (8, 30, 0, 0.7, 40)])
@pytest.mark.parametrize("seed", range(4))
def test_generate_beam_is_beam_search(beams, steps, eos, penalty, n, seed):
    vocab = 24
    prompt = np.random.default_rng(seed).integers(0, vocab, n).tolist()
    eng = StandIn(vocab, 200, hashed_logits(vocab), 256)
    toks, scores = eng.generate_beam(prompt, beams, steps, eos_token_id=eos, length_penalty=penalty, use_prefix=False)
    want, ref = plain_search(eng.logits, prompt, beams, steps, eos, penalty)
    assert [tuple(t.tolist()) for t in toks] == want
    # a step's key is rounded to f32 once, at its distance from the best beam: below 2^6 here, so 40 sums
    # of them are off by at most 40 * 2^6 * 2^-24
    assert np.abs(scores - np.array(ref)).max() <= 40 * 2.0 ** -18
    assert eng.pool.num_free == 200


def test_generate_beam_keeps_long_sums():
    """A thousand tokens: the sum is off by the roundings of single steps, not by those of the sum.

    A step's key is rounded to f32 at its distance from the best beam.  Logits of deviation 0.3 over 24
    tokens: a token of the three best beams has a log-probability above -5 and trails the best beam by
    less than 3, so the key stays below 8, half a step of it is at most 2^-22, of the distance 2^-23: 6 *
    2^-24 a step, below 1000 * 2^-21 in all.
    (Half a step of a sum near -2500 itself is 2^-13.)"""
    vocab, steps = 24, 1000
    eng = StandIn(vocab, 400, hashed_logits(vocab, 0.3), 1100)
    prompt = [1, 2, 3]
    toks, scores = eng.generate_beam(prompt, 3, steps, use_prefix=False, length_penalty=0.0)
    for t, s in zip(toks, scores):
        total, seq = 0.0, tuple(prompt)
        for v in t.tolist():
            x = eng.logits(seq).astype(np.float64)
            total += x[v] - x.max() - math.log(np.exp(x - x.max()).sum())
            seq += (v,)
        assert abs(s - total) <= 1000 * 2.0 ** -21
