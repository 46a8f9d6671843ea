"""GPU: attention through a sliding window with sinks against a plain 64-bit computation."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
PAGE = 16


def ops():
    from higgs_b200 import ops as o
    return o


def make(B, Lq, Hq, Hkv, D, lens, W, sinks, seed=0, qscale=1.5):
    """Inputs whose hidden keys are NaN: the slots no query sees, and a page of NaN that the block
    table names wherever no key of a page is visible."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    rng = np.random.default_rng(seed)
    blocks = max(1, -(-max(lens) // PAGE))
    pages = B * blocks + 1
    k = torch.randn(pages, Hkv, PAGE, D, generator=g, device=DEV).bfloat16()
    v = torch.randn(pages, Hkv, PAGE, D, generator=g, device=DEV).bfloat16()
    q = (qscale * torch.randn(B, Lq, Hq, D, generator=g, device=DEV)).bfloat16()
    ids = rng.permutation(pages)
    poison, bt = int(ids[-1]), ids[:-1].reshape(B, blocks).astype(np.int32).copy()
    seen = np.zeros((pages, PAGE), bool)
    for b, n in enumerate(lens):
        p0 = max(0, n - Lq)
        for pg in range(blocks):
            vis = [j < n and (j >= p0 - W + 1 or j < sinks) for j in range(pg * PAGE, pg * PAGE + PAGE)]
            seen[bt[b, pg]] = vis
            if not any(vis):
                bt[b, pg] = poison
    dead = torch.from_numpy(~seen).to(DEV)[:, None, :, None]
    k.masked_fill_(dead, math.nan)
    v.masked_fill_(dead, math.nan)
    return q, k, v, torch.from_numpy(bt).to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)


def plain(q, k, v, bt, lens, W, sinks, scale=None):
    """(out, sum of weights times |v|) in 64 bits, from the definition."""
    B, Lq, Hq, D = q.shape
    Hkv = k.shape[1]
    scale = 1 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(B, Lq, Hq, D, dtype=torch.float64, device=DEV)
    mag = torch.zeros_like(out)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        ids = bt[b, :-(-n // PAGE)].long()
        kk = k[ids].double().transpose(1, 2).reshape(-1, Hkv, D)[:n].nan_to_num(0.0)
        vv = v[ids].double().transpose(1, 2).reshape(-1, Hkv, D)[:n].nan_to_num(0.0)
        p = (n - Lq + torch.arange(Lq, device=DEV))[:, None]
        j = torch.arange(n, device=DEV)[None]
        see = (j <= p) & ((j > p - W) | (j < sinks))
        for h in range(Hq):
            s = q[b, :, h].double() @ kk[:, h * Hkv // Hq].t() * scale
            s = torch.where(see, s, -math.inf)
            w = torch.where(see, (s - s.amax(1, keepdim=True)).exp(), 0.0)
            w = w / w.sum(1, keepdim=True)
            w = torch.where(see.any(1, keepdim=True), w, 0.0)
            out[b, :, h] = w @ vv[:, h * Hkv // Hq]
            mag[b, :, h] = w @ vv[:, h * Hkv // Hq].abs()
    return out, mag


def check(got, ref, mag, rows):
    """One bf16 rounding of the result (2^-8 of it) and the errors inside, relative to sum w |v|.
    Scores: |q . k| scale stays below 16 here, so f32 products summed over D = 128 are off by at
    most 128 * 2^-23 * 16 < 2^-12, in weight and in norm: 2^-11; exp2 and the 16-bit weights of
    the decode kernel are far below that.  More than 64 query rows per kv head: weights rounded to
    bf16, 2^-8."""
    tol = 2.0 ** -8 * ref.abs() + (2.0 ** -11 + (2.0 ** -8 if rows > 64 else 0.0)) * mag
    err = (got.double() - ref).abs()
    assert torch.isfinite(got).all()
    assert (err <= tol).all(), f"worst {(err / tol.clamp(min=1e-30)).max().item():.3f} of the tolerance"


CASES = [
    # B, Lq, Hq, Hkv, D, lens, window, sinks
    (1, 1, 32, 8, 128, [2048], 1024, 4),
    (4, 1, 32, 8, 128, [700, 33, 1500, 64], 500, 4),
    (3, 1, 8, 2, 64, [0, 1, 17], 1, 0),          # an empty sequence, a window of the key itself
    (3, 1, 7, 1, 128, [500, 33, 90], 16, 100),   # more sinks than window, than some sequences
    (2, 1, 48, 2, 128, [200, 31], 77, 5),        # 24 heads per kv head
    (5, 1, 8, 8, 64, [16, 15, 1000, 48, 0], 31, 16),
    (2, 6, 32, 8, 64, [300, 5], 10, 3),          # fewer keys than queries: rows that see nothing
    (2, 3, 16, 8, 128, [1, 40], 12, 0),
    (1, 9, 40, 8, 128, [640], 20, 17),           # 45 query rows per kv head
    (2, 16, 8, 2, 64, [777, 16], 300, 1),        # 64 query rows
    (2, 70, 6, 2, 64, [400, 69], 33, 16),        # 3 heads per kv head, a row without position
    (1, 300, 8, 8, 128, [300], 128, 0),
    (1, 257, 32, 4, 128, [1000], 2 ** 31 - 1, 0),  # no window: the causal mask
    (2, 130, 14, 2, 128, [900, 0], 1, 2),
    (1, 513, 32, 8, 128, [2100], 250, 130),      # sinks over more than one block of keys
    (3, 40, 16, 4, 64, [2000, 7, 513], 600, 4),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(str(x) for x in c[:5]))
def test_window_attention_vs_plain(case):
    B, Lq, Hq, Hkv, D, lens, W, sinks = case
    q, k, v, bt, sl = make(*case, seed=sum(lens) + Lq)
    got = ops().window_attention(q, k, v, bt, sl, max(max(lens), 1), W, sinks)
    ref, mag = plain(q, k, v, bt, lens, W, sinks)
    check(got, ref, mag, Hq // Hkv * Lq)
    for b, n in enumerate(lens):
        if n < Lq:
            assert (got[b, :Lq - n] == 0).all()
    again = ops().window_attention(q, k, v, bt, sl, max(max(lens), 1), W, sinks)
    assert torch.equal(got, again)


@pytest.mark.parametrize("Lq", [1, 5, 200])
def test_window_wider_than_the_cache_is_paged_attention(Lq):
    lens = [211, 400]
    q, k, v, bt, sl = make(2, Lq, 32, 8, 128, lens, 4096, 0, seed=Lq)
    k, v = k.nan_to_num(0.0), v.nan_to_num(0.0)
    a = ops().window_attention(q, k, v, bt, sl, 400, 4096).float()
    b = ops().paged_attention(q, k, v, bt, sl, 400).float()
    _, mag = plain(q, k, v, bt, lens, 4096, 0)
    # two results, each within one rounding and (above 64 rows) bf16 weights of the exact one
    tol = 2 * (2.0 ** -8 * torch.maximum(a.abs(), b.abs()) + (2.0 ** -11 + (2.0 ** -8 if Lq > 16 else 0)) * mag)
    assert ((a - b).abs() <= tol).all()


@pytest.mark.parametrize("case", [(1, 100, 8, 2, 128, [300], 77, 5), (2, 90, 14, 2, 64, [50, 400], 33, 0)],
                         ids=["d128", "d64"])
def test_window_attention_many_rows_without_tensor_cores(case):
    """The 8-row kernel on prompts (option attn_prefill_tc off): its 16-bit weights, many tiles."""
    from higgs_b200 import ffi
    q, k, v, bt, sl = make(*case, seed=1)
    ffi.call("higgs_set_option", b"attn_prefill_tc", 0)
    try:
        got = ops().window_attention(q, k, v, bt, sl, max(case[5]), case[6], case[7])
    finally:
        ffi.call("higgs_set_option", b"attn_prefill_tc", 1)
    ref, mag = plain(q, k, v, bt, case[5], case[6], case[7])
    check(got, ref, mag, 1)


@pytest.mark.parametrize("Lq", [1, 4, 100])
def test_window_attention_strided_caches(Lq):
    """A layer of a [pages, layers, ...] pool, and a head-major pool: pages and heads by strides."""
    lens = [150, 600]
    q, k, v, bt, sl = make(2, Lq, 16, 4, 64, lens, 90, 4, seed=3)
    want = ops().window_attention(q, k, v, bt, sl, 600, 90, 4)
    big = [torch.stack([torch.full_like(x, math.nan), x], 1) for x in (k, v)]
    assert torch.equal(want, ops().window_attention(q, big[0][:, 1], big[1][:, 1], bt, sl, 600, 90, 4))
    hm = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (k, v)]
    assert torch.equal(want, ops().window_attention(q, hm[0], hm[1], bt, sl, 600, 90, 4))


@pytest.mark.parametrize("Lq", [1, 100])
def test_window_attention_offsets_past_32_bits(Lq):
    """Pages more than 2^32 bytes from the pool's start."""
    D, Hkv, pages = 128, 8, 150000  # 32 KB pages: 4.9 GB
    lens = [100]
    q, k, v, bt, sl = make(1, Lq, 8, Hkv, D, lens, 50, 4, seed=9)
    want = ops().window_attention(q, k, v, bt, sl, 100, 50, 4)
    big = torch.empty(pages, Hkv, PAGE, D, dtype=torch.bfloat16, device=DEV)
    n = k.shape[0]
    big[-n:] = k
    vbig = torch.empty_like(big)
    vbig[-n:] = v
    assert torch.equal(want, ops().window_attention(q, big, vbig, bt + (pages - n), sl, 100, 50, 4))


def test_window_attention_graphs_share_a_workspace():
    """Two captured calls of different shapes over one workspace, replayed in turn while the cache
    grows, on a side stream."""
    o = ops()
    W, sinks = 100, 4
    a = make(2, 1, 32, 8, 128, [400, 390], 100000, sinks, seed=1)
    b = make(1, 200, 8, 2, 64, [300], W, sinks, seed=2)
    ws = torch.zeros(max(x.numel() for x in (
        o.window_attention_workspace(2, 1, 32, 8, 128, 400, W, sinks, DEV),
        o.window_attention_workspace(1, 200, 8, 2, 64, 300, W, sinks, DEV))), dtype=torch.uint8, device=DEV)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    outs, graphs = [], []
    with torch.cuda.stream(st):
        for x, m in ((a, 400), (b, 300)):
            o.window_attention(*x, m, W, sinks, workspace=ws)
            gr = torch.cuda.CUDAGraph()
            st.synchronize()
            with torch.cuda.graph(gr, stream=st):
                outs.append(o.window_attention(*x, m, W, sinks, workspace=ws))
            graphs.append(gr)
        for n in (120, 257, 400):
            a[4].copy_(torch.tensor([n, n - 10], dtype=torch.int32))
            for gr in graphs:
                gr.replay()
            st.synchronize()
            ref, mag = plain(*a[:4], [n, n - 10], W, sinks)
            check(outs[0], ref, mag, 4)
            ref, mag = plain(*b[:4], [300], W, sinks)
            check(outs[1], ref, mag, 800)


def test_window_attention_refuses():
    o = ops()
    from higgs_b200.ffi import HiggsError
    q, k, v, bt, sl = make(2, 1, 8, 2, 64, [40, 30], 16, 0)
    ok = (q, k, v, bt, sl, 40, 16, 0)
    with pytest.raises(HiggsError, match="window >= 1"):
        o.window_attention(q, k, v, bt, sl, 40, 0)
    with pytest.raises(HiggsError, match="sinks >= 0"):
        o.window_attention(q, k, v, bt, sl, 40, 16, -1)
    with pytest.raises(HiggsError, match="block table too short"):
        o.window_attention(q, k, v, bt, sl, 49, 16)
    with pytest.raises(HiggsError, match="workspace too small"):
        o.window_attention(*ok[:5], 48, 48, workspace=torch.zeros(64, dtype=torch.uint8, device=DEV))
    with pytest.raises(TypeError):
        o.window_attention(q.float(), *ok[1:])
    with pytest.raises(TypeError):
        o.window_attention(q, k, v, bt.long(), *ok[4:])
    with pytest.raises(ValueError):
        o.window_attention(q.transpose(0, 2), *ok[1:])
    with pytest.raises(ValueError):
        o.window_attention(q, k, v[:, :1], *ok[3:])
    with pytest.raises(ValueError):
        o.window_attention(q, k, v, bt, sl[:1], *ok[5:])
    with pytest.raises(ValueError):
        o.window_attention(q, k, v, bt.cpu(), *ok[4:])
    with pytest.raises(HiggsError, match="D must be 64 or 128"):
        o.window_attention(q[..., :32].contiguous(), k[..., :32].contiguous(), v[..., :32].contiguous(), *ok[3:])
    with pytest.raises(HiggsError, match="16-byte aligned"):
        o.window_attention(*ok[:5], 40, 16, workspace=torch.zeros(1 << 20, dtype=torch.uint8, device=DEV)[8:])


def test_window_attention_scale_and_sharp_scores():
    """A scale of the caller's, and scores so sharp that one key takes all: the running maximum is
    raised often."""
    for Lq, rows in ((1, 4), (150, 600)):
        q, k, v, bt, sl = make(1, Lq, 8, 2, 128, [700], 500, 4, seed=Lq, qscale=6.0)
        got = ops().window_attention(q, k, v, bt, sl, 700, 500, 4, scale=0.25)
        ref, mag = plain(q, k, v, bt, [700], 500, 4, scale=0.25)
        # scores up to 6 * 4 sigma * sqrt(128) * 0.25 < 2^7 here, so the f32 sums of 128 products are off by
        # at most 128 * 2^-23 * 2^7 = 2^-9 in weight and norm: 2^-8 of sum w |v|; bf16 weights add 2^-8
        tol = 2.0 ** -8 * ref.abs() + (2.0 ** -8 + (2.0 ** -8 if rows > 64 else 0)) * mag
        assert torch.isfinite(got).all() and ((got.double() - ref).abs() <= tol).all()
        for bad in (0.0, -1.0, math.inf, math.nan):
            from higgs_b200.ffi import HiggsError
            with pytest.raises(HiggsError, match="scale"):
                ops().window_attention(q, k, v, bt, sl, 700, 500, 4, scale=bad)


def test_window_attention_default_workspace_on_a_side_stream():
    """Calls on two streams at once, each with a workspace of its own."""
    a = make(2, 1, 32, 8, 128, [900, 333], 256, 4, seed=21)
    b = make(1, 130, 32, 8, 128, [900], 256, 4, seed=22)
    want = [ops().window_attention(*x, 900, 256, 4) for x in (a, b)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for x, st in zip((a, b), streams):
            with torch.cuda.stream(st):
                got.append(ops().window_attention(*x, 900, 256, 4))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert torch.equal(g, want[i % 2])
