"""The operators of long and branching generations, as cases: attention through a sliding window
with sinks over the paged cache, copies of cache pages, and beam search's selection.

``run`` computes a case either with elementary torch operations (``own`` false) or through
``higgs_b200.ops`` (``own`` true); ``exact`` computes it from the definition in 64 bits.
"""
import math

import numpy as np
import torch

own = False

PAGE = 16
DEV = "cuda"


# ---- cases ------------------------------------------------------------------------------------

def _window(name, B, Lq, Hq, Hkv, D, W, sinks, max_len, min_len):
    return {"name": name, "op": "window_attention", "B": B, "Lq": Lq, "Hq": Hq, "Hkv": Hkv, "D": D,
            "W": W, "sinks": sinks, "max_len": max_len, "min_len": min_len}


def _copy(name, kind, layers, Hkv, D, pages, n, fan):
    return {"name": name, "op": "kv_copy_pages", "kind": kind, "layers": layers, "Hkv": Hkv, "D": D,
            "pages": pages, "n": n, "fan": fan}


def _beam(name, B, W, V, n, first=False, masked=False):
    return {"name": name, "op": "beam_select", "B": B, "W": W, "V": V, "n": n, "first": first,
            "masked": masked}


def listed():
    return [
        # one chat decoding with a short window: a latency-bound layer of a 32 / 8-head model
        _window("window_decode_b1", 1, 1, 32, 8, 128, 1024, 4, 2048, 2048),
        # a full batch of long chats, every length another one: the bandwidth-bound decode layer
        _window("window_decode_b32", 32, 1, 32, 8, 128, 4096, 4, 32768, 5000),
        # speculative verify of six tokens with 64-wide heads, lengths shorter than the window too
        _window("window_verify_d64", 8, 6, 32, 8, 64, 1000, 8, 4001, 3),
        # a 2048-token prompt chunk behind a cached prefix, window inside the chunk
        _window("window_prefill_2k", 1, 2048, 32, 8, 128, 1024, 16, 4096, 4096),
        # a whole long prompt, window half of it; the largest attention call
        _window("window_prefill_8k", 1, 8192, 32, 8, 128, 4096, 4, 8192, 8192),
        # four beams fork the page they are filling from two parents
        _copy("copy_fork_4", "bf16", 28, 8, 128, 64, 4, 2),
        # 77 TurboQuant pages (codes and scales of K and V) moved down into holes
        _copy("copy_tq4_77", "tq4", 36, 8, 128, 300, 77, 1),
        # the pool packed after a busy hour: 500 pages of all layers
        _copy("copy_compact_500", "bf16", 36, 8, 128, 1100, 500, 1),
        # one request, four beams, the first step (only beam 0 lives)
        _beam("beam_b1_w4", 1, 4, 128256, 8, first=True),
        # an odd vocabulary (rows that start on no 16-byte boundary), a token mask on it
        _beam("beam_b3_w5_odd", 3, 5, 32003, 10, masked=True),
        # eight requests of eight beams
        _beam("beam_b8_w8", 8, 8, 151936, 16),
        # the largest selection: 32 requests of 16 beams, twice as many candidates
        _beam("beam_b32_w16", 32, 16, 151936, 32),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["window_attention", "window_attention", "kv_copy_pages", "beam_select"])
    top = {k: max(work(c)[k] for c in listed() if c["op"] == op) for k in ("bytes", "flops")}
    while True:
        if op == "window_attention":
            Hkv, G = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 7, 8])
            mode = rng.choice(["decode", "verify", "prefill"])
            Lq = {"decode": 1, "verify": rng.randint(2, 9), "prefill": _log_int(rng, 17, 8192)}[mode]
            B = _log_int(rng, 1, 48) if mode != "prefill" else rng.randint(1, 3)
            top_len = _log_int(rng, max(Lq, 16), 32768)
            c = _window(None, B, Lq, G * Hkv, Hkv, rng.choice([64, 128]), _log_int(rng, 1, 8192),
                        rng.choice([0, 1, 4, 16, 100]), top_len,
                        rng.choice([0, max(1, top_len // 3), top_len]))
            # the plain form holds the scores of one kv head of a sequence in 32 bits
            if Lq * G * (c["W"] + Lq + c["sinks"]) > 5e8:
                continue
        elif op == "kv_copy_pages":
            kind = rng.choice(["bf16", "bf16", "tq4"])
            n = _log_int(rng, 1, 500)
            c = _copy(None, kind, rng.randint(1, 48), rng.choice([1, 2, 3, 4, 8]),
                      128 if kind == "tq4" else rng.choice([64, 128]), 2 * n + rng.randint(1, 100),
                      n, rng.choice([1, 1, 2, 4]))
        else:
            W = rng.randint(1, 16)
            c = _beam(None, _log_int(rng, 1, 32), W, _log_int(rng, 1000, 160000), rng.randint(1, 2 * W),
                      rng.random() < 0.2, rng.random() < 0.3)
        w = work(c)
        if w["bytes"] <= top["bytes"] and w["flops"] <= top["flops"]:
            del c["name"]
            return c


def _lens(c):
    """Cache lengths of a window case: from max_len down to min_len over the batch."""
    B = c["B"]
    if B == 1:
        return [c["max_len"]]
    return [c["max_len"] - (c["max_len"] - c["min_len"]) * b // (B - 1) for b in range(B)]


def work(c):
    if c["op"] == "window_attention":
        keys = pairs = 0
        for n in _lens(c):
            p0 = max(0, n - c["Lq"])  # the first query that has a position
            lo = max(0, p0 - c["W"] + 1)
            keys += max(0, n - lo) + min(c["sinks"], lo, n)
            p = np.arange(p0, n, dtype=np.int64)
            in_win = np.minimum(p + 1, c["W"])
            pairs += int((in_win + np.minimum(c["sinks"], p + 1 - in_win)).sum())
        q = c["B"] * c["Lq"] * c["Hq"] * c["D"]
        return {"bytes": 4 * q + 4 * keys * c["Hkv"] * c["D"], "flops": 4 * pairs * c["Hq"] * c["D"]}
    if c["op"] == "kv_copy_pages":
        page = sum(math.prod(s[2:]) * t.itemsize for s, t in _pools(c))
        srcs = -(-c["n"] // c["fan"])  # each source page is read once
        return {"bytes": c["layers"] * (srcs + c["n"]) * page, "flops": 0}
    logits = c["B"] * c["W"] * c["V"]
    return {"bytes": 4 * logits + 4 * c["B"] * c["W"] + 12 * c["B"] * c["n"], "flops": 3 * logits}


def _pools(c):
    """Shapes and types of a cache: K and V, or their codes and scales."""
    L, P, H = c["layers"], c["pages"], c["Hkv"]
    if c["kind"] == "bf16":
        return [((L, P, H, PAGE, c["D"]), torch.bfloat16)] * 2
    return [((L, P, H, PAGE, c["D"] // 2), torch.uint8), ((L, P, H, PAGE), torch.float16)] * 2


# ---- inputs -----------------------------------------------------------------------------------

def prepare(c, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    rng = np.random.default_rng(seed)
    st = {"case": c}
    if c["op"] == "window_attention":
        B, Hkv, D, lens = c["B"], c["Hkv"], c["D"], _lens(c)
        blocks = max(1, -(-c["max_len"] // PAGE))
        # pages a sequence still owns: those a query of this call can see; the pages between the
        # sinks and the window have been freed (no id in the table)
        own_page = np.zeros((B, blocks), bool)
        for b, n in enumerate(lens):
            lo = max(0, n - c["Lq"] - c["W"] + 1)
            own_page[b, lo // PAGE:-(-n // PAGE)] = True
            own_page[b, :-(-min(c["sinks"], n) // PAGE)] = True
        total = int(own_page.sum())
        pages = total + 3
        bt = np.full((B, blocks), -1, np.int32)
        bt[own_page] = rng.permutation(pages)[:total]
        # normalised and rotated heads: keys of unit variance, queries a little sharper
        st["q"] = (1.5 * torch.randn(B, c["Lq"], c["Hq"], D, generator=g, device=DEV)).bfloat16()
        st["k"] = torch.randn(pages, Hkv, PAGE, D, generator=g, device=DEV).bfloat16()
        st["v"] = torch.randn(pages, Hkv, PAGE, D, generator=g, device=DEV).bfloat16()
        st["bt"] = torch.from_numpy(bt).to(DEV)
        st["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        if own:
            from higgs_b200 import ops
            st["ws"] = ops.window_attention_workspace(B, c["Lq"], c["Hq"], Hkv, D, c["max_len"],
                                                      c["W"], c["sinks"], st["q"].device)
    elif c["op"] == "kv_copy_pages":
        st["pools"] = [torch.randint(0, 256, s, dtype=t, generator=g, device=DEV) if t == torch.uint8
                       else torch.randn(s, generator=g, device=DEV, dtype=t) for s, t in _pools(c)]
        n, fan = c["n"], c["fan"]
        ids = rng.permutation(c["pages"]).astype(np.int32)
        st["dst"] = ids[:n]
        st["src"] = np.repeat(ids[n:n + -(-n // fan)], fan)[:n].copy()
    else:
        B, W, V = c["B"], c["W"], c["V"]
        # beams of one request agree on most of the vocabulary
        x = torch.randn(B, W, V, generator=g, device=DEV)
        x.mul_(0.7).add_(2.5 * torch.randn(B, 1, V, generator=g, device=DEV))
        if c["masked"]:  # a grammar leaves about one token in fifty
            keep = torch.rand(B, W, V, generator=g, device=DEV) < 0.02
            x.masked_fill_(~keep, -math.inf)
        s = torch.randn(B, W, generator=g, device=DEV).abs().mul(-4).sort(1, descending=True).values
        if c["first"]:
            s[:, 1:] = -math.inf
        st["logits"], st["scores"] = x.view(B * W, V), s.contiguous()
        if own:
            from higgs_b200 import ops
            st["ws"] = ops.beam_select_workspace(B, W, V, c["n"], x.device)
    return st


# ---- one pass ---------------------------------------------------------------------------------

def run(st):
    c = st["case"]
    if own:
        from higgs_b200 import ops
        if c["op"] == "window_attention":
            return ops.window_attention(st["q"], st["k"], st["v"], st["bt"], st["lens"], c["max_len"],
                                        c["W"], c["sinks"], workspace=st["ws"])
        if c["op"] == "kv_copy_pages":
            ops.kv_copy_pages(st["pools"], st["src"], st["dst"])
            return st["pools"]
        return ops.beam_select(st["logits"], st["scores"], c["n"], workspace=st["ws"])
    return {"window_attention": _plain_window, "kv_copy_pages": _plain_copy,
            "beam_select": _plain_beam}[c["op"]](st)


def _plain_window(st):
    c, q, lens = st["case"], st["q"], st["lens"].long()
    B, Lq, Hq, Hkv, D, W, sinks = (c[k] for k in ("B", "Lq", "Hq", "Hkv", "D", "W", "sinks"))
    G = Hq // Hkv
    span = min(W + Lq - 1, c["max_len"])
    # the keys some query can see: the first ones, then the last `span` of each sequence
    first = torch.arange(min(sinks, c["max_len"]), device=DEV).expand(B, -1)
    last = lens[:, None] - span + torch.arange(span, device=DEV)
    idx = torch.cat([first, last], 1)
    live = torch.cat([first < lens[:, None], last >= sinks], 1)
    page = st["bt"].long().gather(1, idx.clamp(0, st["bt"].shape[1] * PAGE - 1) // PAGE)
    live &= page >= 0
    p = lens[:, None] - Lq + torch.arange(Lq, device=DEV)
    out = torch.empty(B, Lq, Hq, D, dtype=torch.bfloat16, device=DEV)
    for b in range(B):
        ok = live[b] & (idx[b] <= p[b][:, None]) & ((idx[b] > p[b][:, None] - W) | (idx[b] < sinks))
        k = st["k"][page[b].clamp(0), :, idx[b] % PAGE].float()
        v = st["v"][page[b].clamp(0), :, idx[b] % PAGE].float() * live[b][:, None, None]
        step = max(1, int(6e8) // (G * Lq * idx.shape[1]))  # kv heads at a time
        for h in range(0, Hkv, step):
            kh, vh = k[:, h:h + step].transpose(0, 1), v[:, h:h + step].transpose(0, 1)
            qh = q[b, :, h * G:(h + step) * G].float().view(Lq, -1, G, D).permute(1, 2, 0, 3)
            s = (qh.reshape(len(kh), G * Lq, D) @ kh.transpose(1, 2)) * (1.0 / math.sqrt(D))
            s = s.view(len(kh), G, Lq, -1).masked_fill_(~ok, -math.inf)
            m = s.amax(-1, keepdim=True)
            e = s.sub_(torch.where(m == -math.inf, torch.zeros_like(m), m)).exp_()
            z = e.sum(-1, keepdim=True)
            o = (e.view(len(kh), G * Lq, -1) @ vh).view(len(kh), G, Lq, D)
            o = o / torch.where(z == 0, torch.ones_like(z), z)
            out[b, :, h * G:(h + step) * G] = o.permute(2, 0, 1, 3).reshape(Lq, -1, D).to(torch.bfloat16)
    return out


def _plain_copy(st):
    src = torch.from_numpy(st["src"]).to(DEV).long()
    dst = torch.from_numpy(st["dst"]).to(DEV).long()
    for pool in st["pools"]:
        pool[:, dst] = pool[:, src]
    return st["pools"]


def _plain_beam(st):
    c, x, n = st["case"], st["logits"], st["case"]["n"]
    B, W, V = c["B"], c["W"], c["V"]
    m = x.amax(1, keepdim=True)
    # sums of 64 bits: which of two near candidates wins depends on the difference of two of them
    lse = m.double()[:, 0] + (x - m).exp().sum(1, dtype=torch.float64).log()
    k = min(n, V)
    val, tok = torch.sort(x, dim=1, descending=True, stable=True)
    val, tok = val[:, :k].contiguous(), tok[:, :k].contiguous()
    key = (st["scores"].double().view(-1, 1) - lse[:, None]) + val.double()
    key = torch.where(torch.isnan(key), torch.full_like(key, -math.inf), key).view(B, W * k)
    key, at = torch.sort(key, dim=1, descending=True, stable=True)
    key, at = key[:, :n], at[:, :n]
    if key.shape[1] < n:
        pad = n - key.shape[1]
        key = torch.nn.functional.pad(key, (0, pad), value=-math.inf)
        at = torch.nn.functional.pad(at, (0, pad))
    none = key == -math.inf
    beams = torch.where(none, -1, at // k).int()
    toks = torch.where(none, -1, tok.view(B, W * k).gather(1, at)).int()
    return key.float(), beams, toks


# ---- the definition in 64 bits ----------------------------------------------------------------

def exact(c, seed):
    st = prepare(c, seed)
    return {"window_attention": _exact_window, "kv_copy_pages": _exact_copy,
            "beam_select": _exact_beam}[c["op"]](c, st)


def _exact_window(c, st):
    """Every query against every key position of its sequence, hidden ones included, in blocks of
    queries; hidden positions weigh nothing."""
    G = c["Hq"] // c["Hkv"]
    out = torch.zeros(c["B"], c["Lq"], c["Hq"], c["D"], dtype=torch.float64, device=DEV)
    for b, n in enumerate(_lens(c)):
        if n == 0:
            continue
        ids = st["bt"][b, :-(-n // PAGE)].long()
        kv = []
        for t in ("k", "v"):
            x = torch.zeros(len(ids), c["Hkv"], PAGE, c["D"], dtype=torch.float64, device=DEV)
            x[ids >= 0] = st[t][ids[ids >= 0]].double()
            kv.append(x.permute(1, 0, 2, 3).reshape(c["Hkv"], -1, c["D"])[:, :n])
        j = torch.arange(n, device=DEV)
        step = max(1, int(6e7) // (n * G))
        for t0 in range(0, c["Lq"], step):
            t1 = min(c["Lq"], t0 + step)
            p = (n - c["Lq"] + torch.arange(t0, t1, device=DEV))[:, None]
            see = (j <= p) & ((p - j < c["W"]) | (j < c["sinks"]))
            some = see.any(1)
            if not bool(some.any()):
                continue
            for h in range(c["Hkv"]):
                qh = st["q"][b, t0:t1, h * G:(h + 1) * G].double()
                s = torch.einsum("tgd,jd->gtj", qh, kv[0][h]) / math.sqrt(c["D"])
                w = torch.softmax(torch.where(see, s, -math.inf), -1)
                o = torch.einsum("gtj,jd->tgd", torch.where(see, w, 0.0), kv[1][h])
                out[b, t0:t1, h * G:(h + 1) * G] = torch.where(some[:, None, None], o, 0.0)
    return out


def _exact_copy(c, st):
    want = [p.clone() for p in st["pools"]]
    for s, d in zip(st["src"].tolist(), st["dst"].tolist()):
        for w, p in zip(want, st["pools"]):
            w[:, d].copy_(p[:, s])
    return want


def _exact_beam(c, st):
    B, W, V, n = c["B"], c["W"], c["V"], c["n"]
    vals = torch.full((B, n), -math.inf, dtype=torch.float64)
    beams = torch.full((B, n), -1, dtype=torch.int32)
    toks = torch.full((B, n), -1, dtype=torch.int32)
    for b in range(B):
        x = st["logits"].view(B, W, V)[b].double()
        key = (st["scores"][b].double()[:, None] + torch.log_softmax(x, 1)).reshape(-1)
        key = torch.nan_to_num(key, nan=-math.inf, posinf=math.inf, neginf=-math.inf)
        edge = torch.topk(key, min(n, W * V)).values[-1]
        at = torch.nonzero((key >= edge) & (key > -math.inf))[:, 0].cpu().numpy()
        k = key[torch.from_numpy(at).to(DEV)].cpu().numpy()
        order = np.lexsort((at, -k))[:n]
        m = len(order)
        vals[b, :m] = torch.from_numpy(k[order].copy())
        beams[b, :m] = torch.from_numpy((at[order] // V).astype(np.int32))
        toks[b, :m] = torch.from_numpy((at[order] % V).astype(np.int32))
    return vals.to(DEV), beams.to(DEV), toks.to(DEV)
