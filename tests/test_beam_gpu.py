"""GPU: beam search's selection against a plain 64-bit computation."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def ops():
    from higgs_b200 import ops as o
    return o


def plain(x, s, n):
    """x [B, W, V], s [B, W] -> (keys f64, beams, tokens) [B, n], from the definition."""
    B, W, V = x.shape
    x = np.where(np.isnan(x), -np.inf, x).astype(np.float64)
    keys = np.full((B, n), -np.inf)
    beams, toks = np.full((B, n), -1, np.int32), np.full((B, n), -1, np.int32)
    for b in range(B):
        m = x[b].max(1, keepdims=True)
        live = np.isfinite(m[:, 0]) & np.isfinite(s[b])
        m = np.where(live[:, None], m, 0.0)
        with np.errstate(all="ignore"):
            z = m[:, 0] + np.log(np.exp(x[b] - m).sum(1))
            k = (s[b].astype(np.float64) - z)[:, None] + x[b]
        k = np.where(live[:, None], k, -np.inf).reshape(-1)
        order = np.argsort(-k, kind="stable")[:n]
        order = order[k[order] > -np.inf]
        keys[b, :order.size] = k[order]
        beams[b, :order.size] = order // V
        toks[b, :order.size] = order % V
    return keys, beams, toks


def run(x, s, n, **kw):
    out = ops().beam_select(torch.from_numpy(x.astype(np.float32)).to(DEV), torch.from_numpy(s.astype(np.float32)).to(DEV),
                            n, **kw)
    return [t.cpu().numpy() for t in out]


# Keys: one rounding to f32 (2^-24 of the key) and the log sum: exponentials good to a few ulps
# (2^-21 relative, arguments up to 32: 2^-24 * 32 = 2^-19 only for terms below e^-30 of the sum)
# and tree sums in f32 of 2^13 terms: below 2^-20 of the sum.
def tol(keys):
    k = np.where(np.isfinite(keys), np.abs(keys), 0)
    return 2.0 ** -24 * k + 2.0 ** -20


def check(x, s, n, **kw):
    got = run(x, s, n, **kw)
    keys, beams, toks = plain(x, s.astype(np.float32), n)
    fin = np.isfinite(keys)
    assert (np.isfinite(got[0]) == fin).all()
    assert (np.abs(got[0][fin] - keys[fin]) <= tol(keys)[fin]).all()
    assert np.array_equal(got[1], beams)
    assert np.array_equal(got[2], toks)
    return got


def draw(seed, B, W, V, sd=2.5):
    rng = np.random.default_rng(seed)
    x = (rng.normal(0, sd, (B, 1, V)) + rng.normal(0, 0.7, (B, W, V))).astype(np.float32)
    return x, np.sort(-np.abs(rng.normal(0, 4, (B, W))), 1)[:, ::-1].astype(np.float32).copy()


@pytest.mark.parametrize("B,W,V,n", [(1, 1, 1, 1), (1, 1, 7, 3), (2, 3, 50, 6), (1, 4, 8192, 8), (3, 5, 32003, 10),
                                     (2, 8, 8193, 16), (1, 32, 151936, 32), (4, 1, 163840, 32), (7, 16, 1000, 31),
                                     (300, 2, 257, 4)])
def test_beam_select_vs_plain(B, W, V, n):
    x, s = draw(B + W + V + n, B, W, V)
    check(x, s, n)


def test_beam_select_first_step_and_dead_beams():
    x, s = draw(1, 3, 4, 5000)
    s[:, 1:] = -np.inf
    s[1, 0] = np.nan
    s[2, 3] = -1.0
    got = check(x, s, 8)
    assert (got[1][1] == -1).all() and np.isneginf(got[0][1]).all()


def test_beam_select_more_candidates_than_tokens():
    x, s = draw(2, 2, 3, 5)
    x[0, 1] = -np.inf          # a row without mass
    x[1, :, 1:] = -np.inf      # one token allowed
    x[1, 2, 0] = np.inf        # a row without a log sum
    check(x, s, 16)


def test_beam_select_nan_and_masked_rows():
    x, s = draw(3, 2, 4, 9000)
    rng = np.random.default_rng(4)
    x[rng.random(x.shape) < 0.3] = np.nan
    x[rng.random(x.shape) < 0.9] = -np.inf
    x[1, 2] = np.nan
    check(x, s, 12)


def test_beam_select_lowest_values():
    """Masks of the type's lowest value weigh nothing, but can be chosen when nothing else is left."""
    x, s = draw(5, 1, 2, 4000)
    low = np.finfo(np.float32).min
    x[:, :, 3:] = low
    got = run(x, s, 10)
    keys, beams, toks = plain(x, s, 10)
    assert np.array_equal(got[2][:, :6], toks[:, :6]) and np.array_equal(got[1][:, :6], beams[:, :6])
    assert (got[0][:, 6:] < -1e38).all()  # -inf once rounded past f32's range, or the lowest value


@pytest.mark.parametrize("V", [40, 20000, 20001])
def test_beam_select_ties_go_to_the_lower_index(V):
    """Equal logits within a row, and equal rows with equal scores: beam * V + token decides."""
    x = np.zeros((2, 4, V), np.float32)
    x[1] = np.tile(np.round(np.random.default_rng(V).normal(0, 1, V) * 2) / 2, (4, 1))
    s = np.full((2, 4), -1.5, np.float32)
    check(x, s, 16)


@pytest.mark.parametrize("order", ["rising", "falling", "one_thread"])
def test_beam_select_placement(order):
    """The largest logits next to one another, or all of one thread's."""
    V = 3 * 8192 + 100
    x, s = draw(6, 2, 2, V, sd=1.0)
    if order != "one_thread":
        x = np.sort(x, 2)
        x = x if order == "rising" else x[:, :, ::-1].copy()
    else:
        x[:, :, 77:8192:256] += 20 + np.random.default_rng(7).random(32).astype(np.float32)
        x[:, :, 8192 + 77:16384:256] += 20 + np.random.default_rng(8).random(32).astype(np.float32)
    check(x, s, 32)


def test_beam_select_repeats_and_graph():
    o = ops()
    x, s = draw(9, 4, 4, 30000)
    xt, stt = torch.from_numpy(x).to(DEV), torch.from_numpy(s).to(DEV)
    ws = o.beam_select_workspace(4, 4, 30000, 8, DEV)
    first = o.beam_select(xt, stt, 8, workspace=ws)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, o.beam_select(xt, stt, 8, workspace=ws)))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=st):
            out = o.beam_select(xt, stt, 8, workspace=ws)
        x2, s2 = draw(10, 4, 4, 30000)
        xt.copy_(torch.from_numpy(x2))
        stt.copy_(torch.from_numpy(s2))
        gr.replay()
        gr.replay()
        st.synchronize()
    keys, beams, toks = plain(x2, s2, 8)
    assert np.array_equal(out[1].cpu().numpy(), beams) and np.array_equal(out[2].cpu().numpy(), toks)


def test_beam_select_refuses():
    o = ops()
    from higgs_b200.ffi import HiggsError
    x = torch.zeros(4, 10, device=DEV)
    s = torch.zeros(1, 4, device=DEV)
    for n in (0, 33, -1):
        with pytest.raises(HiggsError, match="n_out"):
            o.beam_select(x, s, n)
    with pytest.raises(HiggsError, match="beams 1..32"):
        o.beam_select(torch.zeros(33, 10, device=DEV), torch.zeros(1, 33, device=DEV), 4)
    with pytest.raises(HiggsError, match="V 1..163840"):
        o.beam_select(torch.zeros(4, 163841, device=DEV), s, 4)
    with pytest.raises(HiggsError, match="workspace too small"):
        o.beam_select(x, s, 4, workspace=torch.zeros(4096, dtype=torch.uint8, device=DEV))
    with pytest.raises(TypeError):
        o.beam_select(x.half(), s, 4)
    with pytest.raises(ValueError):
        o.beam_select(x, torch.zeros(2, 4, device=DEV), 4)
    with pytest.raises(ValueError):
        o.beam_select(x.cpu(), s, 4)


@pytest.mark.parametrize("B,W,V,n", [(1, 16, 151936, 32), (1, 8, 151936, 16), (30, 16, 20000, 32), (445, 1, 9000, 3),
                                     (6, 32, 4096, 32), (1, 2, 4097, 1)])
def test_beam_select_shares_and_lists(B, W, V, n):
    """Shapes of every way the rows are shared out: many lists per request, rows cut across CTAs,
    more rows than CTAs, single rounds."""
    x, s = draw(B + W + V, B, W, V)
    check(x, s, n)


def test_beam_select_many_equal_keys_across_lists():
    """More equal candidates than are ranked directly: every beam alike, few distinct values."""
    V = 40000
    row = np.round(np.random.default_rng(1).normal(0, 1, V) * 4).astype(np.float32) / 4
    x = np.tile(row, (2, 32, 1))
    check(x, np.full((2, 32), -2.0, np.float32), 32)
    check(np.zeros((1, 32, V), np.float32), np.zeros((1, 32), np.float32), 32)


def test_beam_select_unaligned_logits():
    """A row length of a multiple of four on a base that is not 16-byte aligned."""
    x, s = draw(3, 2, 4, 5000)
    buf = torch.empty(2 * 4 * 5000 + 1, device=DEV)
    buf[1:] = torch.from_numpy(x).to(DEV).view(-1)
    got = ops().beam_select(buf[1:].view(8, 5000), torch.from_numpy(s).to(DEV), 8)
    keys, beams, toks = plain(x, s, 8)
    assert np.array_equal(got[1].cpu().numpy(), beams) and np.array_equal(got[2].cpu().numpy(), toks)
    assert (np.abs(got[0].cpu().numpy() - keys) <= tol(keys)).all()


def test_beam_select_two_streams():
    x, s = draw(4, 4, 8, 60000)
    xt, st = torch.from_numpy(x).to(DEV), torch.from_numpy(s).to(DEV)
    want = ops().beam_select(xt, st, 16)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(6):
        for sm in streams:
            with torch.cuda.stream(sm):
                got.append(ops().beam_select(xt, st, 16))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


@pytest.mark.parametrize("B,W,V,n", [(4, 16, 151936, 32), (3, 16, 128256, 32), (2, 16, 151936, 32), (1, 32, 151936, 32),
                                     (7, 32, 100001, 32), (5, 9, 151936, 18)])
@pytest.mark.parametrize("live", [1, 2])
def test_beam_select_few_beams_alive(B, W, V, n, live):
    """The first step of wide beams, and beams that died: many lists, of which fewer than n hold anything."""
    x, s = draw(B + W + V + live, B, W, V)
    s[:, live:] = -np.inf
    x[0, 1:live] = np.nan
    check(x, s, n)


@pytest.mark.parametrize("B,W,V,n,lo,hi", [(1, 8, 151936, 16, 1000, 1200), (2, 16, 151936, 32, 70000, 70033),
                                           (1, 32, 128256, 32, 128255, 128256), (1, 16, 151935, 31, 4090, 4100)])
@pytest.mark.parametrize("seed", [0, 1, 2])
def test_beam_select_neighbouring_tokens_allowed(B, W, V, n, lo, hi, seed):
    """A mask that leaves tokens in one or two places of the vocabulary: most lists are empty."""
    x, s = draw(V + lo + seed, B, W, V)
    x[:, :, :lo] = -np.inf
    x[:, :, hi:] = -np.inf
    check(x, s / 20, n)  # beams of similar scores: each list's best is near the others'


def test_beam_select_many_equal_keys_behind_few_heads():
    """More equal candidates than are ranked directly behind fewer than n lists' best ones."""
    x = np.zeros((1, 20, 4096), np.float32)
    x[:, :, 1000] = 5
    check(x, np.full((1, 20), -1.0, np.float32), 32)


@pytest.mark.parametrize("V", [3 * 4096 + 100, 3 * 4096 + 101])
@pytest.mark.parametrize("thread", [0, 77, 255])
def test_beam_select_all_of_one_thread(V, thread):
    """Every candidate in the logits that one thread of the scan loads: with 16-byte loads four
    neighbours of every 1024, else one of every 256."""
    x, s = draw(V + thread, 2, 2, V, sd=1.0)
    at = np.arange(V)
    mine = (at % 1024) // 4 == thread if V % 4 == 0 else at % 256 == thread
    x[:, :, mine] += 20
    got = check(x, s, 32)
    assert mine[got[2]].all()
