"""CPU: forking and packing pages of the pool, renaming them in the prefix cache, and the refusals of
the device entry points that need no device."""
import ctypes

import numpy as np
import pytest

from higgs_b200.ffi import HiggsError
from higgs_b200.kv import BlockPool, PrefixCache


@pytest.mark.parametrize("length", [0, 1, 15, 16, 17, 32, 47, 48])
def test_fork_shares_whole_pages(length):
    pool = BlockPool(10)
    pages = pool.alloc(3)
    mine, copy = pool.fork(pages, length)
    full = length // 16
    assert mine.size == -(-length // 16)
    assert mine[:full].tolist() == pages[:full].tolist()
    assert [pool.refcount(int(p)) for p in pages] == [2] * full + [1] * (3 - full)
    if length % 16:
        assert copy == (int(pages[full]), int(mine[full])) and copy[1] not in pages.tolist()
        assert pool.refcount(copy[1]) == 1 and pool.num_free == 6
    else:
        assert copy is None and pool.num_free == 7
    pool.release(mine)
    pool.release(pages)
    assert pool.num_free == 10


def test_fork_keeps_given_up_pages_and_is_all_or_nothing():
    pool = BlockPool(4)
    pages = pool.alloc(4)
    pool.release(pages[1:2])
    trimmed = [int(pages[0]), -1, int(pages[2]), int(pages[3])]
    mine, copy = pool.fork(trimmed, 50)
    assert mine[1] == -1 and copy[0] == trimmed[3] and copy[1] == int(pages[1])
    with pytest.raises(HiggsError) as e:
        pool.fork(trimmed, 50)
    assert e.value.code == -7
    assert [pool.refcount(p) for p in trimmed if p >= 0] == [2, 2, 1]
    for bad, n in (([0, 99], 20), ([0, -1], 20), ([0], 20), ([0, 1], -1)):
        with pytest.raises(HiggsError):
            pool.fork(bad, n)


@pytest.mark.parametrize("seed", range(8))
def test_compact_packs_pages(seed):
    rng = np.random.default_rng(seed)
    n = int(rng.integers(1, 60))
    pool = BlockPool(n)
    own = pool.alloc(n)
    content = {int(p): i for i, p in enumerate(own)}
    drop = own[rng.random(n) < 0.5]
    pool.release(drop)
    live = [int(p) for p in own if p not in drop]
    for p in live[::3]:
        pool.retain([p])
    counts = {p: pool.refcount(p) for p in live}
    free = pool.num_free
    src, dst = pool.compact()
    assert not set(src.tolist()) & set(dst.tolist()) and len(set(dst.tolist())) == dst.size
    to = dict(zip(src.tolist(), dst.tolist()))
    moved = {to.get(p, p): content[p] for p in live}
    assert sorted(moved) == list(range(len(live))) and pool.num_free == free
    assert all(pool.refcount(to.get(p, p)) == counts[p] for p in live)
    assert pool.compact()[0].size == 0
    if free:
        assert int(pool.alloc(1)[0]) == len(live)  # the lowest free page comes first


def test_compact_bounded():
    pool = BlockPool(10)
    pages = pool.alloc(10)
    pool.release(pages[:5])
    src, dst = pool.compact(2)
    assert src.tolist() == [9, 8] and dst.tolist() == [0, 1]
    src, dst = pool.compact()
    assert src.tolist() == [7, 6, 5] and dst.tolist() == [2, 3, 4]


def test_prefix_cache_remap():
    pool = BlockPool(20)
    pc = PrefixCache(pool, 4)
    hole = pool.alloc(4)
    pages = pool.alloc(3)
    toks = np.arange(48, dtype=np.int32)
    pc.store(toks, pages)
    pool.release(hole)
    src, dst = pool.compact()
    pc.remap(src, dst)
    to = dict(zip(src.tolist(), dst.tolist()))
    pages = np.array([to.get(int(p), int(p)) for p in pages], np.int32)
    m, got = pc.lookup(toks)
    assert m == 48 and got.tolist() == pages.tolist() and sorted(pages.tolist()) == [0, 1, 2]
    pool.release(got)
    pool.release(pages)
    pc.clear()
    assert pool.num_free == 20
    with pytest.raises(ValueError):
        pc.remap([1, 2], [3])


@pytest.fixture(scope="module")
def lib():
    from higgs_b200 import ffi
    return ffi.load()


def _err(lib):
    return lib.higgs_last_error().decode()


def test_window_attention_arguments_without_device(lib):
    """Shape and alignment checks come before any CUDA call."""
    def call(D=128, Hq=32, Hkv=8, B=1, Lq=1, mb=64, msl=1024, w=128, s=4, sc=0.1, q=4096, ps=16384, wsb=1 << 24,
             ws=4096):
        p = 4096
        return lib.higgs_window_attention(p, q, B, Lq, Hq, Hkv, D, p, p, ps, 2048, p, mb, p, msl, w, s,
                                          ctypes.c_float(sc), p, ws, wsb, None)
    for kw, why in ((dict(D=96), "D must be"), (dict(w=0), "window >= 1"), (dict(s=-1), "sinks >= 0"),
                    (dict(Hq=30), "head shape"), (dict(B=0), "head shape"), (dict(Lq=0), "head shape"),
                    (dict(msl=1025), "block table too short"), (dict(msl=0), "head shape"),
                    (dict(q=4098), "16-byte aligned"), (dict(ps=16385), "16-byte aligned"),
                    (dict(ws=4104), "16-byte aligned"), (dict(sc=0.0), "scale"), (dict(sc=float("nan")), "scale"),
                    (dict(wsb=16), "workspace too small"), (dict(q=None), "null argument")):
        assert call(**kw) in (-1, -4), kw
        assert why in _err(lib), (kw, _err(lib))


@pytest.mark.parametrize("page,head", [(-16384, 2048), (0, 2048), (16384, -2048), (16384, 0)])
def test_window_attention_strides_must_be_positive(lib, page, head):
    for Lq in (1, 100):  # both kernels
        assert lib.higgs_window_attention(4096, 4096, 1, Lq, 32, 8, 128, 4096, 4096, page, head, 4096, 64, 4096, 1024,
                                          128, 4, ctypes.c_float(0.1), 4096, 4096, 1 << 24, None) == -1
        assert "positive" in _err(lib)


def test_window_attention_workspace_size(lib):
    f = lib.higgs_window_attention_workspace_size
    assert f(1, 1, 32, 8, 128, 2048, 1024, 4) > 16384
    assert f(1, 2048, 32, 8, 128, 4096, 1024, 4) == 16384  # tensor-core tiles: counters only
    assert f(1, 1, 32, 8, 128, 2048, 2 ** 31 - 1, 2 ** 31 - 1) == f(1, 1, 32, 8, 128, 2048, 2048, 2048)
    for bad in ((0, 1, 32, 8, 128, 64, 8, 0), (1, 1, 30, 8, 128, 64, 8, 0), (1, 1, 32, 8, 96, 64, 8, 0),
                (1, 1, 32, 8, 128, 64, 0, 0), (1, 1, 32, 8, 128, 64, 8, -1)):
        assert f(*bad) == 0


def test_beam_select_arguments_without_device(lib):
    def call(B=1, W=4, V=1000, n=8, ws=4096, wsb=1 << 24, logits=4096):
        p = 4096
        return lib.higgs_beam_select(p, logits, p, B, W, V, n, p, p, p, ws, wsb, None)
    for kw, why in ((dict(B=0), "B 1..1024"), (dict(B=1025), "B 1..1024"), (dict(W=33), "beams 1..32"),
                    (dict(V=163841), "V 1..163840"), (dict(n=0), "n_out 1..32"), (dict(n=33), "n_out 1..32"),
                    (dict(ws=4100), "16-byte"), (dict(wsb=4607), "workspace too small"), (dict(logits=None), "null")):
        assert call(**kw) in (-1, -4), kw
        assert why in _err(lib), (kw, _err(lib))
    f = lib.higgs_beam_select_workspace_size
    assert f(1, 33, 1000, 4) == 0 and f(1, 4, 1000, 4) > 4096 and f(1024, 32, 163840, 32) > 0


def test_kv_copy_arguments_without_device(lib):
    def call(src, dst, base=4096, layers=1, pages=10, ls=16000, ps=1600, pb=1600, n_pools=1):
        words = (ctypes.c_int64 * 6)(base or 0, layers, pages, ls, ps, pb)
        s, d = np.array(src, np.int32), np.array(dst, np.int32)
        return lib.higgs_kv_copy_pages(4096, words, n_pools, s.ctypes.data, d.ctypes.data, s.size, None)
    assert call([], []) == 0
    for a, kw, why in ((([1, 2], [3, 3]), {}, "two copies"), (([1, 3], [3, 4]), {}, "also a source"),
                       (([1], [1]), {}, "also a source"), (([1], [10]), {}, "outside"), (([-1], [1]), {}, "outside"),
                       (([1], [2]), dict(base=4100), "multiples of 16"), (([1], [2]), dict(pb=1601), "multiples of 16"),
                       (([1], [2]), dict(ps=1584), "overlap"), (([1], [2]), dict(pages=0), "empty pool"),
                       (([1], [2]), dict(base=None), "empty pool"), (([1], [2]), dict(n_pools=0), "1 to 8"),
                       (([1], [2]), dict(n_pools=9), "1 to 8")):
        assert call(*a, **kw) == -1, (a, kw)
        assert why in _err(lib), (a, kw, _err(lib))


def test_set_attention_window_without_device(lib):
    assert lib.higgs_model_set_attention_window(None, 16, 0) == -1
    assert "bad argument" in _err(lib)


def _engine_whose_copies_fail(pages=12):
    from higgs_b200.engine import Engine
    eng = Engine.__new__(Engine)
    eng.pool = BlockPool(pages)

    def fail(src, dst):
        raise RuntimeError("copy")
    eng._copy_pages = fail
    return eng


def test_forks_give_their_pages_back_when_the_copy_fails():
    from higgs_b200.engine import Sequence
    eng = _engine_whose_copies_fail()
    seq = Sequence(prompt=np.zeros(20, np.int32), pages=eng.pool.alloc(2).tolist(), length=20)
    with pytest.raises(RuntimeError):
        eng.fork(seq, 3)
    assert eng.pool.num_free == 10 and [eng.pool.refcount(p) for p in seq.pages] == [1, 1]
    with pytest.raises(RuntimeError):
        eng._reorder([seq], [(0, 1, 0.0), (0, 2, 0.0), (0, 3, 0.0)])
    assert eng.pool.num_free == 10 and [eng.pool.refcount(p) for p in seq.pages] == [1, 1]
    eng.release(seq)
    assert eng.pool.num_free == 12


def test_kv_copy_refuses_overlapping_layers(lib):
    """Layers apart, or interleaved within a page's stride; nothing that would race."""
    def call(layers, pages, layer_stride, page_stride, page_bytes=64):
        words = (ctypes.c_int64 * 6)(4096, layers, pages, layer_stride, page_stride, page_bytes)
        return lib.higgs_kv_copy_pages(4096, words, 1, 4096, 4096, 0, None)
    assert call(3, 10, 640, 64) == 0     # [layers, pages]
    assert call(3, 10, 64, 192) == 0     # [pages, layers]
    assert call(1, 10, 0, 64) == 0       # one layer: its stride is not used
    assert call(3, 1, 64, 0) == 0        # one page: nor is the pages'
    for bad in ((3, 10, 0, 64), (3, 10, 576, 64), (3, 10, 64, 176), (3, 10, 48, 192), (2, 10, -640, 64),
                (2, 2 ** 62, 64, 64), (2, 10, 64, 2 ** 62)):
        rc = call(*bad)
        assert rc == (0 if bad == (2, 10, 64, 2 ** 62) else -1), bad
        if rc:
            assert "overlap" in _err(lib), bad


def test_sizes_past_32_bits_are_refused_not_cut():
    """A size that does not fit the C interface's ints must not arrive as its lower half."""
    import torch

    from higgs_b200 import ops
    from higgs_b200.model import Model, tiny_args
    big = 2 ** 32 + 5
    q = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16)
    kv = torch.zeros(4, 1, 16, 64, dtype=torch.bfloat16)
    bt, sl = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for args in ((big, 16, 0), (64, big, 0), (64, 16, big), (64, -big, 0), (64, 16, -big)):
        with pytest.raises(ValueError, match="32 bits"):
            ops.window_attention(q, kv, kv, bt, sl, *args)
        with pytest.raises(ValueError, match="32 bits"):
            ops.window_attention_workspace(1, 1, 2, 1, 64, *args, "cpu")
    with pytest.raises(ValueError, match="32 bits"):
        ops.beam_select(torch.zeros(2, 8), torch.zeros(1, 2), big)
    with pytest.raises(ValueError, match="32 bits"):
        ops.beam_select_workspace(1, 2, 8, big, "cpu")
    for kw in (dict(attn_window=big), dict(attn_window=8, attn_sinks=big)):
        with pytest.raises(ValueError, match="32 bits"):
            Model(tiny_args("qwen3", 1), {}, num_pages=4, **kw)
    pool = BlockPool(4)
    with pytest.raises(ValueError, match="32 bits"):
        pool.fork(pool.alloc(1), big)
    src, _ = pool.compact(big)  # more than there are pages: all
    assert src.size == 0
    pool.alloc(1)
    pool.release([0])
    assert [x.tolist() for x in pool.compact(big)] == [[1], [0]]


def test_compact_changes_nothing_when_the_copy_fails():
    from higgs_b200.engine import Sequence
    eng = _engine_whose_copies_fail()
    eng.prefix = PrefixCache(eng.pool, 4)
    hole = eng.pool.alloc(3)
    seq = Sequence(prompt=np.zeros(40, np.int32), pages=eng.pool.alloc(3).tolist(), length=40)
    toks = np.arange(32, dtype=np.int32)
    eng.prefix.store(toks, np.array(seq.pages[:2], np.int32))
    eng.pool.release(hole)
    pages = list(seq.pages)
    with pytest.raises(RuntimeError):
        eng.compact([seq])
    assert seq.pages == pages and [eng.pool.refcount(p) for p in pages] == [2, 2, 1]
    assert eng.pool.num_free == 9 and eng.prefix.lookup(toks)[1].tolist() == pages[:2]
    eng.pool.release(pages[:2])
    eng.release(seq)  # the pages are still this sequence's
    eng.prefix.clear()
    assert eng.pool.num_free == 12


def test_pool_move_takes_compaction_back_and_refuses():
    pool = BlockPool(6)
    pages = pool.alloc(6)
    pool.retain(pages[5:])
    pool.release(pages[:2])
    src, dst = pool.compact()
    pool.move(dst, src)
    assert [pool.refcount(p) for p in range(6)] == [0, 0, 1, 1, 1, 2] and pool.num_free == 2
    for s, d in (([2, 0], [1, 3]), ([2, 3], [0, 0]), ([2, 2], [0, 1]), ([0], [1]), ([6], [0]), ([-1], [0]), ([2], [6])):
        with pytest.raises(HiggsError):
            pool.move(s, d)
        assert [pool.refcount(p) for p in range(6)] == [0, 0, 1, 1, 1, 2]
    with pytest.raises(ValueError):
        pool.move([2], [0, 1])
    assert pool.alloc(2).tolist() == [0, 1]


def test_compact_refuses_when_a_sequence_is_missing():
    """A sequence that is not named would keep the old ids of its moved pages."""
    from higgs_b200.engine import Sequence
    eng = _engine_whose_copies_fail()
    eng._copy_pages = lambda src, dst: None
    eng.prefix = PrefixCache(eng.pool, 4)
    hole = eng.pool.alloc(2)
    a, b = (Sequence(prompt=np.zeros(40, np.int32), pages=eng.pool.alloc(3).tolist(), length=40) for _ in range(2))
    toks = np.arange(32, dtype=np.int32)
    eng.prefix.store(toks, np.array(a.pages[:2], np.int32))
    eng.prefix.store(np.concatenate([toks, toks]), np.array(a.pages[:2] + b.pages[:2], np.int32))
    assert eng.prefix.uses(a.pages + b.pages + [99]).tolist() == [2, 2, 0, 1, 1, 0, 0]
    shared = Sequence(prompt=a.prompt, pages=list(a.pages), length=40)
    eng.pool.retain(a.pages)
    eng.pool.release(hole)
    before = [list(a.pages), list(b.pages), [eng.pool.refcount(p) for p in range(12)]]
    for seqs in ([], [a], [a, b][:1], [a, shared]):
        with pytest.raises(ValueError, match="owners"):
            eng.compact(seqs)
        assert before == [a.pages, b.pages, [eng.pool.refcount(p) for p in range(12)]]
    assert eng.compact([a, b, shared, a]) == 2  # a sequence named twice is one
    assert sorted(a.pages + b.pages) == list(range(6)) and shared.pages == a.pages
    for s in (a, b, shared):
        eng.release(s)
    eng.prefix.clear()
    assert eng.pool.num_free == 12


def test_speculative_steps_give_up_pages_behind_the_window():
    """A windowed model's pages behind the window go back to the pool at speculative steps too, and the
    slots and lengths of the step stay those of the untrimmed sequence."""
    import types

    import torch

    from higgs_b200.engine import Engine, Sequence, SpecDecoder
    B, k, pages = 2, 3, 40

    def staged(window, lengths):
        eng = Engine.__new__(Engine)
        eng.pool = BlockPool(pages)
        eng.model = types.SimpleNamespace(attn_window=window, attn_sinks=4)
        dec = SpecDecoder.__new__(SpecDecoder)
        dec.engine, dec.B, dec.k = eng, B, k
        n = 4 * k * B + 3 * B * (k + 1) + B + 2 * k * B + B
        dec.step_host, dec.step_dev = (torch.zeros(n, dtype=torch.int32) for _ in range(2))
        dec.block_table = torch.zeros(B, 20, dtype=torch.int32)
        dec.bt_host = np.zeros((B, 20), np.int32)
        dec.tok = torch.zeros(k + 1, B, dtype=torch.int32)
        seqs = [Sequence(prompt=np.zeros(1, np.int32), length=n, last_token=1) for n in lengths]
        for s in seqs:
            eng._ensure_pages(s, s.length)
        steps = []
        for it in range(12):
            dec.stage(seqs, np.zeros(2 * k * B + B, np.float32), first=it == 0)
            steps.append([[s.length, [s.pages[(s.length + i) // 16] >= 0 for i in range(k + 1)]] for s in seqs])
            for s in seqs:
                s.length += 3
        return eng, seqs, steps

    eng, seqs, steps = staged(24, [90, 7])
    _, _, want = staged(0, [90, 7])
    assert steps == want and all(all(x[1]) for st in steps for x in st)
    # 123 + 4 tokens: page 0 (sinks) and those from key 123 - 23 on, 40 + 4: page 0 and from key 17 on
    assert [[i for i, p in enumerate(s.pages) if p >= 0] for s in seqs] == [[0, 6, 7], [0, 1, 2]]
    assert eng.pool.num_free == pages - 6
    for s in seqs:
        eng.release(s)
    assert eng.pool.num_free == pages
