"""GPU: copies of cache pages, byte for byte."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def ops():
    from higgs_b200 import ops as o
    return o


def pools(kind, layers, pages, Hkv, D, seed=0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    if kind == "bf16":
        shapes = [((layers, pages, Hkv, 16, D), torch.bfloat16)] * 2
    else:
        shapes = [((layers, pages, Hkv, 16, D // 2), torch.uint8), ((layers, pages, Hkv, 16), torch.float16)] * 2
    # random bytes: NaN patterns too
    return [torch.randint(-2 ** 15, 2 ** 15, s[:-1] + (s[-1] * t.itemsize // 2,), dtype=torch.int16, generator=g,
                          device=DEV).view(t).view(s) for s, t in shapes]


def bits(t):
    return t.contiguous().view(torch.int16)


def check(ps, src, dst):
    want = [p.clone() for p in ps]
    for s, d in zip(src, dst):
        for w, p in zip(want, ps):
            w[:, int(d)] = p[:, int(s)]
    ops().kv_copy_pages(ps, src, dst)
    for w, p in zip(want, ps):
        assert torch.equal(bits(w), bits(p))


@pytest.mark.parametrize("kind,layers,Hkv,D", [("bf16", 3, 8, 128), ("bf16", 1, 1, 64), ("bf16", 2, 3, 64),
                                               ("tq4", 3, 8, 128), ("tq4", 2, 1, 128), ("tq4", 5, 3, 128)])
@pytest.mark.parametrize("n", [1, 16, 17, 128, 129])
def test_kv_copy_pages(kind, layers, Hkv, D, n):
    ids = np.random.default_rng(n).permutation(2 * n + 3)
    check(pools(kind, layers, 2 * n + 3, Hkv, D, seed=n), ids[:n], ids[n:2 * n])


def test_kv_copy_pages_more_than_one_launch():
    ids = np.random.default_rng(1).permutation(5000)
    check(pools("tq4", 2, 5000, 1, 128), ids[:2400], ids[2400:4800])


def test_kv_copy_pages_one_source_many_destinations():
    check(pools("bf16", 4, 40, 2, 128), [7] * 20 + [3] * 5, list(range(10, 30)) + list(range(30, 35)))


def test_kv_copy_pages_strided_pool():
    """[pages, layers, ...]: the layers' pages interleaved in memory; and a pool of one layer."""
    ps = [p.transpose(0, 1).contiguous().transpose(0, 1) for p in pools("bf16", 3, 20, 2, 64)]
    check(ps, [1, 5, 9], [0, 19, 2])
    check([p[1:2] for p in pools("bf16", 3, 20, 2, 64)], [4], [3])


def test_kv_copy_pages_past_32_bits():
    p = torch.zeros(1, 150000, 8, 16, 128, dtype=torch.bfloat16, device=DEV)  # 4.9 GB
    p[0, 3] = 2.0
    p[0, 149999] = 3.0
    ops().kv_copy_pages([p], [3, 149999], [149998, 0])
    assert (p[0, 149998] == 2).all() and (p[0, 0] == 3).all() and (p[0, 1] == 0).all()


def test_kv_copy_pages_graph_and_stream():
    ps = pools("bf16", 2, 10, 2, 64)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    src, dst = np.array([1, 2]), np.array([8, 9])
    with torch.cuda.stream(st):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=st):
            ops().kv_copy_pages(ps, src, dst)
        src[:], dst[:] = 0, [3, 4]  # the graph keeps the lists it was captured with
        for p in ps:
            p[:, 1] = 5
        gr.replay()
        st.synchronize()
    for p in ps:
        assert (p[:, 8] == 5).all() and torch.equal(bits(p[:, 9]), bits(p[:, 2]))


def test_kv_copy_pages_empty_and_refusals():
    o = ops()
    from higgs_b200.ffi import HiggsError
    ps = pools("bf16", 2, 10, 2, 64)
    before = [p.clone() for p in ps]
    o.kv_copy_pages(ps, [], [])
    for src, dst, why in (([1, 2], [3, 3], "two copies"), ([1, 3], [3, 4], "also a source"), ([1], [1], "also a source"),
                          ([1], [10], "outside"), ([-1], [2], "outside"), ([10], [2], "outside")):
        with pytest.raises(HiggsError, match=why):
            o.kv_copy_pages(ps, src, dst)
    with pytest.raises(ValueError):
        o.kv_copy_pages(ps, [1], [2, 3])
    with pytest.raises(ValueError):
        o.kv_copy_pages([], [1], [2])
    with pytest.raises(ValueError):
        o.kv_copy_pages([p[..., :32] for p in ps], [1], [2])
    with pytest.raises(HiggsError, match="multiples of 16"):
        o.kv_copy_pages([torch.zeros(1, 4, 5, dtype=torch.bfloat16, device=DEV)], [1], [2])
    with pytest.raises(HiggsError, match="1 to 8 pools"):
        o.kv_copy_pages(ps * 5, [1], [2])
    for a, b in zip(before, ps):
        assert torch.equal(bits(a), bits(b))
