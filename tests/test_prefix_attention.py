"""Attention of sequences that share prefixes (shared_prefix_attention).

GPU: the kernels against the oracle (oracle/block.py), which puts each sequence's slots behind its prefix's, with the
bounds of the paged attention's tests: scores are float32 sums of D products (off by D + 8 half steps of float32 of the
largest sum of |q k|), the softmax weights are rounded to the operands' type for their product with V (half a step of each, in
the sum of p |v|), the output once more. CPU: refusals and what watches operators, with the oracle in place of the launches.
"""
import ctypes
import math

import pytest
import torch

from oracle import block as ob
from oracle import streaming as st

F32 = 2.0 ** -24
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
MUST_NOT_BE_READ = 2


def _caches(dev, P, B, Hk, D, dtype, pages, prefixes, lengths, seed=0, one_pool=False):
    """(prefix, cache): pages in mixed order; every slot that is in use by none is NaN."""
    from dmad_amd import PagedKVCache

    g = torch.Generator().manual_seed(seed)
    page_p, page_o = pages
    Mp, Mo = max(1, -(-max(prefixes) // page_p)), max(1, -(-max(lengths) // page_o))
    Np, No = P * Mp + MUST_NOT_BE_READ, B * Mo + MUST_NOT_BE_READ
    if one_pool:
        assert page_p == page_o
        at = torch.randperm(Np + No, generator=g).to(torch.int32)
        pools = [[torch.full((Np + No, Hk, page_p, D), math.nan, dtype=dtype) for _ in range(2)]] * 2
        tables = at[:P * Mp].view(P, Mp), at[P * Mp:P * Mp + B * Mo].view(B, Mo)
    else:
        pools = [[torch.full((n, Hk, page, D), math.nan, dtype=dtype) for _ in range(2)] for n, page in ((Np, page_p), (No, page_o))]
        tables = tuple(torch.randperm(n, generator=g)[:b * m].view(b, m).to(torch.int32) for n, b, m in ((Np, P, Mp), (No, B, Mo)))
    for (k_pages, v_pages), table, lens, page in zip(pools, tables, (prefixes, lengths), pages):
        for b, n in enumerate(lens):
            for j in range(-(-n // page)):
                m = min(page, n - j * page)
                for t, sd in ((k_pages, 1.5), (v_pages, 1.0)):
                    t[int(table[b, j]), :, :m] = (torch.randn(Hk, m, D, generator=g) * sd).to(dtype)
    if one_pool:
        k, v = (t.to(dev) for t in pools[0])
        pools = [[k, v]] * 2
    out = []
    for (k, v), table, lens in zip(pools, tables, (prefixes, lengths)):
        n = torch.tensor(lens, dtype=torch.int32).to(dev)
        out.append(PagedKVCache(k.to(dev), v.to(dev), table.contiguous().to(dev), n, n.clone()))
    return out


def _fields(c):
    return {n: getattr(c, n) for n in ("k_pages", "v_pages", "page_table", "lengths")}


def _check(got, ref, dtype, D):
    o, lse = got
    ro, rlse, (pv, sv, size) = ref
    u = torch.finfo(dtype).eps / 2
    es = (D + 8) * F32 * size + 64 * F32 * (1 + rlse.transpose(1, 2)[..., None].abs().nan_to_num(0, posinf=0))
    tol = (u * (1 + 1e-3) + 2 * es) * pv + u * (1 + 1e-3) * ro.abs() + 1e-30
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25 * (sv + 1)
    assert torch.isfinite(o).all()
    err = (o.double() - ro).abs()
    print(f"  o: {float((err / tol).max()):.2f} of its bound", flush=True)
    assert (err <= tol).all()
    none = torch.isinf(rlse)
    assert torch.equal(lse == -math.inf, none)
    assert ((lse.double() - rlse).abs()[~none] <= es.amax(-1).transpose(1, 2)[~none]).all()


def _queries(dev, B, S, Hq, D, dtype, seed=1):
    return (torch.randn(B, S, Hq, D, generator=torch.Generator().manual_seed(seed)) * 1.5).to(dtype).to(dev)


CASES = [
    # P, B, S, Hq, Hk, D, dtype, pages, prefixes, lengths, causal
    (1, 1, 1, 1, 1, 128, "bf16", (16, 16), [1], [1], False),
    (1, 3, 1, 2, 2, 64, "fp16", (16, 16), [257], [1, 0, 17], False),
    (2, 4, 1, 4, 1, 128, "bf16", (16, 48), [40, 0], [3, 0, 0, 65], False),
    (1, 4, 1, 12, 12, 64, "fp16", (64, 16), [900], [64, 1, 30, 7], False),
    (1, 2, 3, 6, 3, 32, "bf16", (32, 32), [129], [3, 95], True),
    (3, 6, 2, 8, 2, 16, "fp16", (16, 16), [100, 33, 7], [2, 2, 9, 40, 17, 3], True),
    (1, 8, 4, 16, 2, 128, "bf16", (64, 64), [1000], [4, 5, 60, 64, 65, 300, 7, 8], True),
    (1, 70, 1, 2, 1, 128, "bf16", (16, 16), [300], [(7 * i) % 61 for i in range(70)], False),
    (2, 20, 7, 8, 2, 128, "fp16", (16, 64), [500, 1], [7 + i for i in range(20)], True),
    (1, 33, 1, 5, 5, 256, "bf16", (16, 16), [260], [1 + i for i in range(33)], False),
    (1, 9, 5, 16, 1, 64, "bf16", (128, 16), [700], [5 * i for i in range(1, 10)], True),
    (1, 40, 2, 8, 1, 64, "fp16", (16, 16), [33], [i for i in range(40)], False),
    (1, 12, 1, 64, 2, 32, "fp16", (16, 16), [600], [2] * 12, False),
    (1, 64, 4, 8, 2, 128, "bf16", (64, 16), [2000], [4 + 3 * i for i in range(64)], True),
    (4, 64, 1, 32, 4, 128, "fp16", (48, 16), [129, 128, 127, 1000], [(11 * i) % 90 for i in range(64)], False),
    (1, 300, 1, 2, 2, 128, "bf16", (16, 16), [97], [1] * 300, False),
    # 16 and 17 rows per key head, behind each head dim
    (1, 16, 1, 3, 3, 128, "fp16", (16, 16), [400], [11 * i for i in range(16)], False),
    (1, 17, 1, 3, 3, 128, "bf16", (16, 16), [400], [11 * i for i in range(17)], False),
    (1, 17, 1, 3, 3, 64, "fp16", (32, 16), [190], [140 - i for i in range(17)], False),
    (1, 17, 1, 2, 2, 256, "fp16", (16, 64), [410], [1] * 17, False),
    (1, 16, 1, 2, 2, 256, "bf16", (16, 64), [410], [150] * 16, False),
    (1, 17, 1, 2, 2, 16, "bf16", (16, 16), [300], [3] * 17, False),
    # own slots of more than 16 rows, in several pieces, behind a prefix of one step
    (1, 3, 20, 4, 2, 128, "bf16", (16, 16), [400], [20, 300, 77], True),
    (1, 2, 1, 40, 2, 64, "fp16", (16, 16), [5], [3000, 2500], False),
    (2, 4, 3, 12, 2, 256, "bf16", (16, 16), [31, 0], [3, 500, 0, 129], False),
    # own slots of more than 32 rows, seen by all of them and causal
    (1, 2, 40, 4, 2, 128, "bf16", (16, 16), [400], [700, 40], False),
    (1, 2, 40, 4, 2, 128, "bf16", (16, 16), [400], [700, 40], True),
    (2, 4, 33, 1, 1, 64, "fp16", (32, 16), [100, 17], [33, 150, 64, 1000], False),
    (1, 3, 1, 136, 2, 256, "bf16", (16, 64), [90], [0, 1, 200], False),
    (1, 5, 150, 2, 2, 128, "fp16", (64, 16), [0], [150, 151, 1200, 160, 300], False),
    # pieces of more than 32 steps
    (1, 17, 1, 64, 64, 128, "bf16", (64, 16), [5003], [1 + i for i in range(17)], False),
    (1, 20, 1, 64, 64, 64, "fp16", (16, 16), [9000], [2 * i for i in range(20)], False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("P,B,S,Hq,Hk,D,dtype,pages,prefixes,lengths,causal", CASES)
def test_attention(gpu, P, B, S, Hq, Hk, D, dtype, pages, prefixes, lengths, causal):
    from dmad_amd import shared_prefix_attention

    print(f"case prefix P={P} B={B} S={S} Hq={Hq} Hk={Hk} D={D} {dtype} {pages} {prefixes} {lengths[:4]} causal={causal}", flush=True)
    t = DTYPES[dtype]
    prefix, cache = _caches(gpu, P, B, Hk, D, t, pages, prefixes, lengths, seed=D + S)
    q = _queries(gpu, B, S, Hq, D, t)
    got = shared_prefix_attention(q, prefix, cache, causal=causal, return_lse=True)
    torch.cuda.synchronize()
    _check(got, ob.prefix_attend(_fields(prefix), _fields(cache), q, causal=causal), t, D)
    # the same again bit for bit, and without lse
    assert torch.equal(shared_prefix_attention(q, prefix, cache, causal=causal), got[0])


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hk,D,S,B", [(4, 2, 64, 1, 3), (16, 2, 128, 4, 12)])
def test_equals_caches_with_the_prefix_in_front(gpu, Hq, Hk, D, S, B):
    """One pool, and page tables that begin with the prefix's pages: what paged_attention gives for them, within the
    rounding of both."""
    from dmad_amd import PagedKVCache, paged_attention, shared_prefix_attention

    t = torch.bfloat16
    lengths = [S + 5 * i for i in range(B)]
    prefix, cache = _caches(gpu, 1, B, Hk, D, t, (16, 16), [320], lengths, seed=5, one_pool=True)
    q = _queries(gpu, B, S, Hq, D, t)
    table = torch.cat((prefix.page_table.expand(B, -1), cache.page_table), 1).contiguous()
    n = cache.lengths + 320
    whole = PagedKVCache(cache.k_pages, cache.v_pages, table, n, n.clone())
    for causal in (False, True):
        o, lse = shared_prefix_attention(q, prefix, cache, causal=causal, return_lse=True)
        r, rl = paged_attention(q, whole, causal=causal, return_lse=True)
        ref = ob.prefix_attend(_fields(prefix), _fields(cache), q, causal=causal)
        _check((o, lse), ref, t, D)
        _check((r, rl), ref, t, D)


@pytest.mark.gpu
@pytest.mark.parametrize("B,Hq", [(4, 4), (48, 8)])
def test_missing_pages_odd_lengths_and_scales(gpu, B, Hq):
    """Pages of -1 and beyond the pool, in prefix and cache, hide their slots; lengths are clipped; nothing seen at all
    gives o = 0, lse = -inf; any scale."""
    from dmad_amd import shared_prefix_attention

    for t in (torch.bfloat16, torch.float16):
        prefix, cache = _caches(gpu, 2, B, 2, 128, t, (16, 16), [200, 70], [(5 * i) % 40 for i in range(B)], seed=9)
        q = _queries(gpu, B, 1, Hq, 128, t)
        prefix.page_table[0, 3] = -1
        prefix.page_table[0, 5] = 10 ** 6
        cache.page_table[1, 0] = -7
        for scale in (1e-3, None, 20.0):
            got = shared_prefix_attention(q, prefix, cache, sm_scale=scale, return_lse=True)
            _check(got, ob.prefix_attend(_fields(prefix), _fields(cache), q, scale=scale), t, 128)
        prefix.page_table[1] = -1
        cache.lengths[B // 2:] = -5
        o, lse = shared_prefix_attention(q, prefix, cache, return_lse=True)
        assert (o[B // 2:] == 0).all() and (lse[B // 2:] == -math.inf).all()
        _check((o, lse), ob.prefix_attend(_fields(prefix), _fields(cache), q), t, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,Hq", [(4, 2, 4), (40, 4, 8)])
def test_what_is_not_seen_does_not_reach(gpu, B, S, Hq):
    """An infinity or NaN in a prefix reaches that prefix's sequences and its key head, one in a sequence's own slots that
    sequence's tokens that see it, one in a query its own row; everything else is bit for bit as without."""
    from dmad_amd import shared_prefix_attention

    t = torch.bfloat16
    prefix, cache = _caches(gpu, 2, B, 2, 128, t, (16, 16), [300, 260], [S + i % 30 for i in range(B)], seed=12)
    q = _queries(gpu, B, S, Hq, 128, t)
    clean = shared_prefix_attention(q, prefix, cache, causal=True)
    half, n = Hq // 2, B // 2
    for where, value in (("k_pages", math.nan), ("v_pages", math.inf), ("v_pages", math.nan)):
        at = (int(prefix.page_table[0, 4]), 1, 3)
        keep = getattr(prefix, where)[at].clone()
        getattr(prefix, where)[at] = value
        o = shared_prefix_attention(q, prefix, cache, causal=True)
        assert not torch.isfinite(o[:n, :, half:]).any(), where
        assert torch.equal(o[:n, :, :half], clean[:n, :, :half]) and torch.equal(o[n:], clean[n:])
        getattr(prefix, where)[at] = keep
        b, slot = 1, int(cache.lengths[1]) - 1  # the last token's own slot
        at = (int(cache.page_table[b, slot // 16]), 0, slot % 16)
        keep = getattr(cache, where)[at].clone()
        getattr(cache, where)[at] = value
        o = shared_prefix_attention(q, prefix, cache, causal=True)
        assert not torch.isfinite(o[b, S - 1, :half]).any()
        assert torch.equal(o[b, :S - 1], clean[b, :S - 1]) and torch.equal(o[b, :, half:], clean[b, :, half:])
        others = [i for i in range(B) if i != b]
        assert torch.equal(o[others], clean[others])
        getattr(cache, where)[at] = keep
    for value in (math.nan, math.inf):
        bad = q.clone()
        bad[2, 0, 1] = value
        o = shared_prefix_attention(bad, prefix, cache, causal=True)
        assert not torch.isfinite(o[2, 0, 1]).any()
        o[2, 0, 1] = clean[2, 0, 1]
        assert torch.equal(o, clean)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_a_sequence_does_not_depend_on_its_neighbours(gpu, dtype, D):
    """Scores that grow along the prefix, so that every row's running maximum moves many times, each row's at slots of its
    own: with other queries beside it a sequence's output stays bit for bit what it is."""
    from dmad_amd import shared_prefix_attention

    t, B, n = DTYPES[dtype], 40, 2000
    prefix, cache = _caches(gpu, 1, B, 2, D, t, (16, 16), [n], [1 + i % 5 for i in range(B)], seed=17)
    slots = torch.arange(prefix.capacity, device=gpu).view(-1, 1, 16).expand(-1, 2, -1)
    prefix.k_pages[prefix.page_table[0].long(), ..., 0] = (slots * (320.0 / n)).to(t)
    q = _queries(gpu, B, 1, 4, D, t)
    # scores that grow by up to 200 over the prefix, by 0.3 to 13 over a tile of 128 slots; a maximum may lag by 5.5
    q[..., 0] = torch.arange(1, B + 1, device=gpu).view(B, 1, 1).to(t) * 0.25
    want = shared_prefix_attention(q, prefix, cache, sm_scale=1 / 16, return_lse=True)
    _check(want, ob.prefix_attend(_fields(prefix), _fields(cache), q, scale=1 / 16), t, D)
    other = q.clone()
    other[1::2, ..., 0] *= 1.7
    other[3::4, ..., 1:] = 0.0
    got = shared_prefix_attention(other, prefix, cache, sm_scale=1 / 16, return_lse=True)
    for a, b in zip(got, want):
        assert torch.equal(a[::2], b[::2])
        assert not torch.equal(a[1::2], b[1::2])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("B,Hq", [(2, 2), (64, 8)])
def test_low_and_heavy_scores(gpu, dtype, B, Hq):
    """All scores very low; and one slot far above all others, which are many: the light ones keep their share."""
    from dmad_amd import shared_prefix_attention

    t = DTYPES[dtype]
    prefix, cache = _caches(gpu, 1, B, 2, 64, t, (16, 16), [1500], [1 + i % 20 for i in range(B)], seed=13)
    q = torch.full((B, 1, Hq, 64), -30.0, dtype=t, device=gpu)
    keep = prefix.k_pages.clone()
    prefix.k_pages[prefix.page_table[0].long()] = 30.0
    ref = ob.prefix_attend(_fields(prefix), _fields(cache), q)
    _check(shared_prefix_attention(q, prefix, cache, return_lse=True), ref, t, 64)
    prefix.k_pages.copy_(keep)
    # one prefix slot 12 above the rest in natural log, its value small
    q = torch.zeros(B, 1, Hq, 64, dtype=t, device=gpu)
    q[..., 0] = 4.0
    prefix.k_pages[..., 0] = 0.0
    at = (int(prefix.page_table[0, 70]), slice(None), 5)
    prefix.k_pages[at][..., 0] = 24.0
    prefix.v_pages[at] = 2.0 ** -14
    _check(shared_prefix_attention(q, prefix, cache, return_lse=True), ob.prefix_attend(_fields(prefix), _fields(cache), q), t, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("B", [4, 40])
def test_pages_beyond_32_bits(gpu, B):
    """Pages at the far end of pools of more than 2^31 elements: bit for bit what small pools give."""
    from dmad_amd import PagedKVCache, shared_prefix_attention

    t, Hk, D, page = torch.bfloat16, 8, 128, 16
    prefix, cache = _caches(gpu, 1, B, Hk, D, t, (page, page), [700], [3 + 5 * i for i in range(B)], seed=2, one_pool=True)
    q = _queries(gpu, B, 1, 16, D, t)
    want = shared_prefix_attention(q, prefix, cache, return_lse=True)
    n, far = prefix.k_pages.shape[0], 132000
    assert far * Hk * page * D > 2 ** 31
    pools = []
    for small in (prefix.k_pages, prefix.v_pages):
        pool = torch.empty(far + n, Hk, page, D, device=gpu, dtype=t)
        pool[:n] = math.nan
        pool[far:] = small
        pools.append(pool)
    moved = [PagedKVCache(*pools, c.page_table + far, c.lengths, c.seen) for c in (prefix, cache)]
    got = shared_prefix_attention(q, *moved, return_lse=True)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_strided_queries(gpu):
    from dmad_amd import shared_prefix_attention

    prefix, cache = _caches(gpu, 1, 4, 2, 64, torch.bfloat16, (32, 16), [70], [3, 9, 20, 5], seed=21)
    g = torch.Generator().manual_seed(22)
    qkv = torch.randn(4, 3, 8, 64, generator=g).to(torch.bfloat16).to(gpu)
    q = qkv[:, :, :4]
    want = shared_prefix_attention(q.contiguous(), prefix, cache, causal=True)
    assert torch.equal(shared_prefix_attention(q, prefix, cache, causal=True), want)
    assert torch.equal(shared_prefix_attention(q.transpose(1, 2).contiguous().transpose(1, 2), prefix, cache, causal=True), want)
    assert torch.equal(shared_prefix_attention(q.transpose(0, 1).contiguous().transpose(0, 1), prefix, cache, causal=True), want)
    flat = torch.zeros(4 * 3 * 4 * 64 + 1, device=gpu, dtype=torch.bfloat16)
    flat[1:] = q.reshape(-1)
    assert torch.equal(shared_prefix_attention(flat[1:].view(4, 3, 4, 64), prefix, cache, causal=True), want)
    one = q[:, :1].expand(4, 3, 4, 64)
    assert torch.equal(shared_prefix_attention(one, prefix, cache), shared_prefix_attention(one.contiguous(), prefix, cache))


@pytest.mark.gpu
@pytest.mark.parametrize("B,Hq", [(3, 8), (48, 16)])
def test_captured_steps_and_two_streams(gpu, B, Hq):
    """A captured step follows lengths, page tables and queries; two graphs and two streams do not disturb each other."""
    from dmad_amd import shared_prefix_attention

    t = torch.bfloat16
    prefix, cache = _caches(gpu, 1, B, 2, 128, t, (16, 16), [400], [40] * B, seed=30)
    lengths = cache.lengths.clone()
    qs = [_queries(gpu, B, 2, Hq, 128, t, seed=i) for i in range(2)]
    outs, graphs = [], []
    for q in qs:
        shared_prefix_attention(q, prefix, cache, causal=True)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(shared_prefix_attention(q, prefix, cache, causal=True, return_lse=True))
        graphs.append(graph)
    for i in range(4):
        cache.lengths.copy_(lengths - 7 * i)
        prefix.lengths.fill_(400 - 130 * i)
        for q in qs:
            q.mul_(-0.9)
        want = [shared_prefix_attention(q, prefix, cache, causal=True, return_lse=True) for q in qs]
        junk = torch.randn(1024, 1024, device=gpu)
        (junk @ junk).sum().item()
        for graph in graphs:
            graph.replay()
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        there = []
        for s, q in zip(streams, qs):
            with torch.cuda.stream(s):
                there.append(shared_prefix_attention(q, prefix, cache, causal=True, return_lse=True))
        torch.cuda.synchronize()
        for got in (outs, there):
            for a, b in zip(got, want):
                assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.gpu
def test_no_sequences_or_tokens(gpu):
    from dmad_amd import PagedKVCache, shared_prefix_attention

    prefix = PagedKVCache.allocate(1, 32, 2, 64, device=gpu, page_size=16)
    cache = PagedKVCache.allocate(3, 32, 2, 64, device=gpu, page_size=16)
    o, lse = shared_prefix_attention(torch.zeros(3, 0, 4, 64, device=gpu, dtype=torch.bfloat16), prefix, cache, return_lse=True)
    assert o.shape == (3, 0, 4, 64) and lse.shape == (3, 4, 0)
    o, lse = shared_prefix_attention(torch.ones(3, 1, 4, 64, device=gpu, dtype=torch.bfloat16), prefix, cache, return_lse=True)
    assert (o == 0).all() and (lse == -math.inf).all()


# ---------------------------------------------------------------- refusals


def _mock(monkeypatch):
    from dmad_amd import kv_cache

    def attend(q, prefix, cache, scale, causal):
        for c in (prefix, cache):
            for n in ("k_pages", "v_pages", "page_table", "lengths"):
                t = getattr(c, n)
                assert t.data_ptr() and not t.is_neg()
        assert q.data_ptr() and not q.is_neg(), "a tensor whose memory does not hold its values"
        o, lse, _ = ob.prefix_attend(_fields(prefix), _fields(cache), q, scale=scale, causal=causal)
        return o.to(q.dtype), lse.float()

    monkeypatch.setattr(kv_cache, "_check_same_device", lambda op, *ts: ts[0].device)
    monkeypatch.setattr(kv_cache, "_prefix_attend", attend)


BOTH = pytest.mark.parametrize("device", ["cpu", pytest.param("gpu", marks=pytest.mark.gpu)])


def _small(request, monkeypatch, device):
    if device == "cpu":
        _mock(monkeypatch)
    dev = request.getfixturevalue("gpu") if device == "gpu" else torch.device("cpu")
    prefix, cache = _caches(dev, 1, 2, 2, 16, torch.bfloat16, (16, 16), [20], [5, 9], seed=3)
    return prefix, cache, _queries(dev, 2, 2, 4, 16, torch.bfloat16)


@BOTH
def test_refusals(request, monkeypatch, device):
    from dmad_amd import PagedKVCache, shared_prefix_attention

    prefix, cache, q = _small(request, monkeypatch, device)
    dev = q.device

    def like(P, Hk, D, dtype=torch.bfloat16):
        return PagedKVCache.allocate(P, 32, Hk, D, dtype, dev, page_size=16)

    bad = [
        (TypeError, "prefix must be", q, None, cache, {}),
        (TypeError, "cache must be", q, prefix, {}, {}),
        (ValueError, "share 2 prefixes evenly", q[:1].expand(3, 2, 4, 16), like(2, 2, 16), like(3, 2, 16), {}),
        (ValueError, "the prefix holds", q, like(1, 1, 16), cache, {}),
        (ValueError, "the prefix holds", q, like(1, 2, 32), cache, {}),
        (ValueError, "the prefix holds", q, like(1, 2, 16, torch.float16), cache, {}),
        (ValueError, "q must be", q[0], prefix, cache, {}),
        (ValueError, "q must be", q[..., :8], prefix, cache, {}),
        (ValueError, "q is", q.half(), prefix, cache, {}),
        (ValueError, "not a multiple", q[:, :, :3], prefix, cache, {}),
        (NotImplementedError, "sm_scale", q, prefix, cache, dict(sm_scale=0.0)),
        (NotImplementedError, "sm_scale", q, prefix, cache, dict(sm_scale=math.inf)),
    ]
    for error, match, qq, p, c, how in bad:
        with pytest.raises(error, match=match):
            shared_prefix_attention(qq, p, c, **how)
    for t in (q, prefix.k_pages, cache.v_pages):
        t.requires_grad_(True)
        with pytest.raises(RuntimeError, match="no backward"):
            shared_prefix_attention(q, prefix, cache)
        with torch.no_grad():
            shared_prefix_attention(q, prefix, cache)
        t.requires_grad_(False)
    with torch.no_grad(), torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(q, torch.ones_like(q))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            shared_prefix_attention(dual, prefix, cache)


@BOTH
def test_negated_views_and_replaced_memory(request, monkeypatch, device):
    from dmad_amd import shared_prefix_attention

    prefix, cache, q = _small(request, monkeypatch, device)
    want = shared_prefix_attention(-q, prefix, cache, causal=True)
    assert torch.equal(shared_prefix_attention(torch._neg_view(q), prefix, cache, causal=True), want)
    was = prefix.v_pages.clone()
    prefix.v_pages.data = was * 2
    cache.v_pages.data = cache.v_pages.data * 2
    assert torch.equal(shared_prefix_attention(-q, prefix, cache, causal=True), want * 2)


@BOTH
@pytest.mark.parametrize("how", ["dispatch mode", "profiled", "compiled", "inference"])
def test_op_and_direct_calls_agree_bitwise(request, monkeypatch, device, how):
    from torch.utils._python_dispatch import TorchDispatchMode

    from dmad_amd import shared_prefix_attention

    names = []

    class Names(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            names.append(str(func))
            return func(*args, **(kwargs or {}))

    prefix, cache, q = _small(request, monkeypatch, device)

    def call(q):
        return shared_prefix_attention(q, prefix, cache, causal=True, return_lse=True)

    want = call(q)
    if how == "dispatch mode":
        with Names():
            got = call(q)
        assert [n for n in names if "dmad" in n] == ["dmad.prefix_attn.default"]
    elif how == "profiled":
        with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as p:
            got = call(q)
        assert "dmad::prefix_attn" in {e.key for e in p.key_averages()}
    elif how == "compiled":
        with torch.no_grad():
            got = torch.compile(lambda q, p, c: shared_prefix_attention(q, p, c, causal=True, return_lse=True), fullgraph=True,
                                backend="aot_eager")(q, prefix, cache)
    else:
        with torch.inference_mode():
            got = call(q)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_registered_op_does_what_it_declares(gpu, request, monkeypatch):
    prefix, cache, q = _small(request, monkeypatch, "gpu")
    f = lambda c: [getattr(c, n) for n in ("k_pages", "v_pages", "page_table", "lengths", "seen")]  # noqa: E731
    torch.library.opcheck(torch.ops.dmad.prefix_attn.default, (q, 0.25, True, *f(prefix), *f(cache)))
    with pytest.raises(ValueError, match="the prefix holds"):
        torch.ops.dmad.prefix_attn(q, 0.25, True, prefix.k_pages[:, :1], prefix.v_pages[:, :1], *f(prefix)[2:], *f(cache))


def test_c_entry_rejects_bad_arguments():
    from dmad_amd import _native as nat

    lib, p, n = nat.lib(), ctypes.c_void_p, ctypes.c_size_t(0)

    def cache(batch=4, heads=2, dim=64, pages=8, **over):
        c = nat.KvCache(16, heads, 16, dim, batch, pages, 256, 256, (ctypes.c_int64 * 3)(heads * 16 * dim, 16 * dim, dim),
                        (ctypes.c_int64 * 3)(heads * 16 * dim, 16 * dim, dim), 256, pages, 256, 256, None, None)
        for k, v in over.items():
            setattr(c, k, v)
        return c

    def size(a, b, S=1, Hq=4):
        return lib.dmad_prefix_attn_workspace_bytes(ctypes.byref(a), ctypes.byref(b), S, Hq, ctypes.byref(n))

    assert size(cache(1), cache()) == 0 and n.value > 0
    need = n.value
    assert size(cache(0), cache()) == 1 and b"evenly" in lib.dmad_last_error()
    assert size(cache(3), cache()) == 1 and size(cache(1, heads=1), cache()) == 1 and size(cache(1, dim=32), cache()) == 1
    assert size(cache(1), cache(), Hq=3) == 1 and size(cache(1), cache(), S=-1) == 1
    assert size(cache(1), cache(), S=1 << 30) == 2
    assert size(cache(1, pages=1 << 20, page_size=1 << 20), cache()) == 2
    st4 = (ctypes.c_int64 * 4)

    def call(S=1, q=256, qs=(256, 256, 64, 1), scale=0.1, o=256, lse=256, ws=256, size=1 << 30, dtype=0, prefix=None):
        return lib.dmad_prefix_attn(dtype, ctypes.byref(prefix or cache(1)), ctypes.byref(cache()), S, 4, p(q), st4(*qs), 0, scale, p(o),
                                    p(lse), p(ws), size, p(0))

    assert call(q=0) == 1 and call(o=0) == 1 and call(lse=0) == 1 and call(q=264) == 1 and call(o=264) == 1
    assert call(scale=0.0) == 2 and call(dtype=2) == 2
    assert call(ws=0) == 3 and call(size=need - 1) == 3 and call(ws=264) == 3
    assert call(S=2, qs=(1024, 256, 64, 1)) == 1 and b"follow one another" in lib.dmad_last_error()
    assert call(prefix=cache(1, k_pages=None)) == 1
