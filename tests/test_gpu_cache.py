"""The paged cache's operators on the GPU against plain forms in 64 bits (tests/cache_oracle.py, which derives the tolerances)."""
import math
import random

import pytest
import torch

from tests import cache_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _clean_status():
    from htree_b200 import ops
    yield
    torch.cuda.synchronize()
    ops.check_status()


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def make(dt, N, H, Hkv, K, V, page, lengths, seed=0, spare=2):
    """q, k, v, caches (pages in random order; what no request holds is NaN), table, lengths."""
    g = torch.Generator(device=DEV).manual_seed(seed + 7 * N + K)
    B = len(lengths)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV, dtype=torch.float32).to(dt)      # noqa: E731
    need = [-(-x // page) for x in lengths]
    P, M = sum(need) + spare, max(max(need), 1) + 1
    ids = torch.randperm(P, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((B, M), -1, dtype=torch.int32)
    kc = torch.full((P, page, Hkv, K), math.nan, dtype=dt, device=DEV)
    vc = torch.full((P, page, Hkv, V), math.nan, dtype=dt, device=DEV)
    for b, n in enumerate(need):
        for j in range(n):
            table[b, j] = i = ids.pop()
            some = min(page, lengths[b] - j * page)
            kc[i, :some], vc[i, :some] = rnd(some, Hkv, K), rnd(some, Hkv, V)
    return dict(q=rnd(B, N, H, K), k=rnd(B, N, Hkv, K), v=rnd(B, N, Hkv, V), k_cache=kc, v_cache=vc, block_table=table.to(DEV), lengths=_ints(lengths))


def tree(B, N, seed=0, pad=0.0):
    rng = random.Random(seed)
    return _ints([[-2 if rng.random() < pad else rng.randint(-1, i - 1) for i in range(N)] for _ in range(B)])


def agrees(s, parents=None, scale=None, out=None):
    import htree_b200 as ht
    got = ht.draft_attention(**s, parents=parents, scale=scale, return_lse=True) if out is None else out
    ref, lse, tol, ltol = oracle.attention(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["block_table"], s["lengths"], parents, scale)
    o, l = got[0].double().cpu(), got[1].double().cpu()
    assert got[0].dtype == s["q"].dtype and got[1].dtype == torch.float32
    empty = lse == -math.inf
    assert torch.equal(l[empty], lse[empty]) and torch.equal(o[empty], ref[empty])
    off, loff = (o - ref).abs() - tol, (l - lse)[~empty].abs() - ltol[~empty]
    assert (off <= 0).all(), f"out off by up to {(o - ref).abs().max():.3g}, {off.max():.3g} above the bound"
    assert (loff <= 0).all(), f"lse off: {loff.max():.3g} above the bound"
    return got


CASES = [
    # dt, N, H, Hkv, K, V, page, lengths, tree, pad
    (FP, 1, 8, 2, 64, 64, 16, [130], False, 0), (FP, 5, 4, 4, 32, 32, 16, [0, 63, 64, 65], True, 0), (FP, 70, 2, 1, 128, 64, 24, [200], False, 0),
    (FP, 3, 5, 1, 256, 256, 8, [7, 129], True, 0.5), (FP, 67, 6, 3, 40, 136, 1, [1, 30], True, 0.2),
    (BF, 1, 16, 1, 128, 128, 16, [1000, 1, 0, 64], False, 0), (BF, 1, 32, 2, 128, 128, 64, [5000], False, 0),
    (BF, 8, 8, 8, 128, 128, 32, [333, 32], True, 0), (BF, 13, 16, 2, 64, 64, 16, [401, 3, 77, 250, 128], True, 0.3),
    (BF, 64, 8, 1, 128, 128, 16, [191, 192], True, 0), (BF, 65, 4, 2, 96, 80, 7, [100, 13], True, 0.1), (BF, 130, 16, 1, 128, 128, 64, [300, 0], False, 0),
    (HF, 2, 4, 2, 32, 32, 256, [511, 512], True, 0), (HF, 9, 10, 2, 64, 128, 16, [65, 700], True, 0.2), (HF, 33, 12, 1, 128, 64, 5, [66], False, 0),
    (HF, 200, 3, 1, 64, 64, 16, [64, 190], True, 0.1), (HF, 1, 1, 1, 8, 8, 3, [5], False, 0), (BF, 4, 6, 2, 256, 192, 16, [140, 20], True, 0),
    (HF, 17, 40, 8, 80, 80, 16, [129, 64, 31], True, 0),
    # 33 to 600 query rows: one and two halves of 128, ends inside a tile and inside a box of a page, several row tiles
    (BF, 33, 1, 1, 64, 64, 16, [127, 128, 129], True, 0.1), (BF, 3, 16, 1, 128, 128, 128, [384, 385], True, 0), (HF, 5, 60, 2, 128, 64, 64, [200, 640, 0], True, 0.3),
    (BF, 8, 32, 2, 64, 128, 32, [1000, 31], True, 0), (HF, 16, 32, 2, 96, 80, 48, [256, 100], True, 0), (BF, 43, 12, 2, 128, 128, 256, [700], False, 0),
    (BF, 257, 4, 2, 128, 128, 16, [140, 3], False, 0), (HF, 600, 1, 1, 64, 64, 16, [0, 300], False, 0), (BF, 40, 16, 2, 128, 128, 7, [90], True, 0.2),
    (BF, 144, 8, 1, 128, 128, 64, [128], True, 0.05), (HF, 20, 14, 2, 32, 96, 16, [333, 16], True, 0.9),
    # fp32 with more than four rows of every width, and a 16-bit group that no box of heads fits
    (FP, 4, 12, 1, 128, 128, 16, [70, 33], True, 0), (FP, 9, 4, 2, 64, 128, 5, [40], True, 0.2), (FP, 17, 8, 1, 64, 64, 16, [1000], False, 0),
    (FP, 2, 2, 1, 96, 40, 16, [129, 0], True, 0), (BF, 30, 9, 3, 128, 128, 32, [260], True, 0.1),
    # rows wider than 128, keys and values of different widths among them, in few and many parts
    (BF, 1, 8, 1, 256, 256, 16, [3000, 17], False, 0), (HF, 1, 4, 2, 192, 128, 64, [640], False, 0), (BF, 7, 10, 2, 136, 256, 5, [300, 0], True, 0.2),
    (HF, 40, 6, 2, 8, 248, 16, [77], True, 0.1), (FP, 1, 4, 1, 256, 256, 16, [2000, 3], False, 0), (FP, 2, 2, 1, 144, 8, 3, [250], True, 0),
    (FP, 3, 10, 2, 200, 256, 16, [500], True, 0.2), (FP, 11, 2, 2, 16, 256, 1, [100, 40], False, 0), (FP, 40, 2, 1, 256, 192, 32, [333], True, 0.1),
    # fp32 with more than sixteen rows: parts of one and of several row tiles of 64
    (FP, 64, 1, 1, 128, 128, 64, [1000, 64], True, 0), (FP, 130, 2, 1, 64, 64, 16, [129, 0, 500], False, 0), (FP, 70, 3, 1, 96, 128, 7, [260], True, 0.3),
    (FP, 20, 8, 2, 32, 24, 16, [63, 65], True, 0.5), (FP, 300, 4, 4, 128, 128, 16, [40], False, 0),
    # ... and with five to eight
    (FP, 1, 7, 1, 128, 128, 16, [1000, 5], False, 0), (FP, 8, 2, 2, 64, 64, 16, [300], True, 0.1), (FP, 2, 6, 2, 256, 144, 8, [222], False, 0),
    (FP, 5, 1, 1, 128, 40, 3, [64, 130], True, 0), (FP, 4, 2, 1, 24, 128, 64, [700], True, 0),
]


@pytest.mark.parametrize("dt,N,H,Hkv,K,V,page,lengths,is_tree,pad", CASES)
def test_attention(dt, N, H, Hkv, K, V, page, lengths, is_tree, pad):
    s = make(dt, N, H, Hkv, K, V, page, lengths)
    agrees(s, tree(len(lengths), N, pad=pad) if is_tree else None)


@pytest.mark.parametrize("dt", [FP, BF, HF])
def test_attention_of_many_splits_and_requests(dt):
    agrees(make(dt, 1, 4, 1, 64, 64, 16, [20000], seed=3))                                       # one unit over all blocks
    agrees(make(dt, 2, 4, 2, 64, 64, 16, [(37 * i) % 300 for i in range(300)], seed=4), tree(300, 2))   # more requests than threads of a warp
    agrees(make(dt, 5, 8, 1, 64, 64, 16, [(91 * i) % 900 for i in range(150)], seed=5), tree(150, 5))
    agrees(make(dt, 3, 40, 2, 128, 128, 16, [2500, 10, 1300], seed=6), tree(3, 3))
    wide = make(dt, 3, 16, 2, 64, 64, 16, [100, 40], seed=7)                                     # a table of many more columns than are held
    wide["block_table"] = torch.cat([wide["block_table"], torch.full((2, 1000), -1, dtype=torch.int32, device=DEV)], 1)
    agrees(wide, tree(2, 3))


@pytest.mark.parametrize("dt,scale", [(FP, 1.0), (BF, 2.0), (HF, -0.3), (BF, 0.0)])
def test_scales(dt, scale):
    agrees(make(dt, 20, 8, 2, 64, 64, 16, [150, 64]), tree(2, 20), scale)


@pytest.mark.parametrize("dt", [FP, BF, HF])
def test_a_chain_is_a_tree(dt):
    import htree_b200 as ht
    s = make(dt, 37, 4, 1, 64, 64, 16, [50, 3])
    chain = _ints([[i - 1 for i in range(37)]] * 2)
    assert torch.equal(ht.draft_attention(**s), ht.draft_attention(**s, parents=chain))


@pytest.mark.parametrize("dt", [FP, BF, HF])
def test_large_scores(dt):
    """One key far above the others, in the middle of the cache and among the drafts; all keys far below zero."""
    s = make(dt, 6, 4, 2, 64, 64, 16, [300, 150])
    s["k_cache"][s["block_table"][0, 7].long()] *= 30
    s["k"][1, 2] *= 30
    agrees(s, tree(2, 6))
    s["q"] = torch.ones_like(s["q"])
    s["k"], s["k_cache"] = -s["k"].abs() * 20, -s["k_cache"].abs() * 20
    agrees(s, tree(2, 6))


@pytest.mark.parametrize("dt", [FP, BF, HF])
@pytest.mark.parametrize("N,K", [(5, 64), (70, 128), (40, 128)])
def test_what_a_draft_does_not_read_does_not_reach_it(dt, N, K):
    """Infinities and NaN in the keys and values of drafts: outputs of those that read them are not finite, all others as if they were not there."""
    import htree_b200 as ht
    s = make(dt, N, 16, 2, K, K, 16, [100, 0])
    par = tree(2, N, seed=5, pad=0.1)
    par[:, 0] = -1
    bad = [1, N // 2, N - 1]
    clean = ht.draft_attention(**s, parents=par, return_lse=True)
    reads = torch.stack([oracle.sees(par[b].tolist(), N)[:, bad].any(1) for b in range(2)]).to(DEV)
    for name, x in (("v", math.nan), ("v", math.inf), ("k", math.nan), ("k", -math.inf)):
        t = dict(s, **{name: s[name].clone()})
        t[name][:, bad, :, ::3] = x
        out, lse = ht.draft_attention(**t, parents=par, return_lse=True)
        assert torch.equal(out[~reads], clean[0][~reads]) and torch.equal(lse[~reads], clean[1][~reads])
        real = reads & (par >= -1)
        if not (name == "k" and x == -math.inf):                 # (a score of NaN or of minus infinity, by the signs of q)
            assert not torch.isfinite(out[real]).all(-1).any()


@pytest.mark.parametrize("dt", [FP, BF, HF])
@pytest.mark.parametrize("N,G,K,lengths", [(13, 8, 64, [200, 128, 0]), (5, 2, 128, [65, 17, 300]), (40, 4, 128, [130, 9, 256]), (150, 2, 64, [70, 0, 128])])
def test_padding_holds_anything(dt, N, G, K, lengths):
    """Drafts that are none (parents below -1), inside and behind the others: NaN and infinity in their q, k and v reach nobody, their children included."""
    import htree_b200 as ht
    s = make(dt, N, 2 * G, 2, K, K, 16, lengths)
    parents = tree(len(lengths), N, seed=5, pad=0.2)
    parents[1, N // 2:] = -2
    pad = parents < -1
    clean = ht.draft_attention(**s, parents=parents, return_lse=True)
    agrees(s, parents, out=clean)
    for name, value in (("q", math.nan), ("k", math.inf), ("v", math.nan), ("v", -math.inf)):
        s[name] = torch.where(pad[:, :, None, None], torch.full_like(s[name], value), s[name])
        out, lse = ht.draft_attention(**s, parents=parents, return_lse=True)
        assert torch.equal(out, clean[0]) and torch.equal(lse, clean[1])


@pytest.mark.parametrize("dt,K", [(FP, 64), (BF, 128), (HF, 64), (BF, 256)])
def test_strides(dt, K):
    """q, k, v as slices of one projection; the cache as [pages, heads, 2, page, width]; a table with more columns than are passed."""
    import htree_b200 as ht
    s = make(dt, 9, 8, 2, K, K, 16, [100, 37])
    plain = ht.draft_attention(**s, parents=tree(2, 9), return_lse=True)
    qkv = torch.cat([s["q"], s["k"], s["v"]], 2)
    both = torch.stack([s["k_cache"].transpose(1, 2), s["v_cache"].transpose(1, 2)], 2).contiguous()
    wide = torch.cat([s["block_table"], torch.full_like(s["block_table"], 1 << 20)], 1)
    t = dict(q=qkv[:, :, :8], k=qkv[:, :, 8:10], v=qkv[:, :, 10:], k_cache=both[:, :, 0].transpose(1, 2), v_cache=both[:, :, 1].transpose(1, 2),
             block_table=wide[:, :s["block_table"].shape[1]], lengths=s["lengths"])
    for a, b in zip(plain, ht.draft_attention(**t, parents=tree(2, 9), return_lse=True)):
        assert torch.equal(a, b)
    # heads that share one row (expanded), rows that do not start on 16 bytes (copied)
    e = dict(s, k=s["k"][:, :, :1].expand(-1, -1, 2, -1), v=s["v"][:1].expand(2, -1, -1, -1))
    f = dict(e, k=e["k"].contiguous(), v=e["v"].contiguous())
    odd = torch.empty(s["q"].numel() + 1, dtype=dt, device=DEV)[1:].view(s["q"].shape).copy_(s["q"])
    assert torch.equal(ht.draft_attention(**e), ht.draft_attention(**f))
    assert torch.equal(ht.draft_attention(**dict(s, q=odd)), ht.draft_attention(**s))


def test_offsets_beyond_32_bits():
    import htree_b200 as ht
    pages, page, D = 70000, 256, 128                        # 2.3e9 elements
    small = make(BF, 2, 4, 1, D, D, page, [1000])
    kc, vc = (torch.zeros(pages, page, 1, D, dtype=BF, device=DEV) for _ in range(2))
    used = small["block_table"][0, :4].long()
    far = torch.arange(pages - 4, pages, device=DEV)
    kc[far], vc[far] = small["k_cache"][used], small["v_cache"][used]
    big = dict(small, k_cache=kc, v_cache=vc, block_table=small["block_table"].clone())
    big["block_table"][0, :4] = far.int()
    assert torch.equal(ht.draft_attention(**big), ht.draft_attention(**small))
    k, v = ht.cache_gather(kc, vc, big["block_table"], big["lengths"], 1000)
    assert torch.equal(k[0], oracle.cached_rows(small["k_cache"], small["block_table"][0], 1000)[0])
    slots = (far[:1] * page + 7).view(1, 1)
    ht.cache_append(small["k"][:, :1], small["v"][:, :1], kc, vc, slots)
    assert torch.equal(kc[far[0], 7], small["k"][0, 0]) and torch.equal(vc[far[0], 7], small["v"][0, 0])


@pytest.mark.parametrize("dt", [FP, BF])
def test_pages_outside_the_cache_are_left_out_and_reported(dt):
    import htree_b200 as ht
    from htree_b200 import ops
    s = make(dt, 3, 8, 2, 64, 64, 16, [100, 90])
    s["block_table"][0, 2], s["block_table"][1, 0] = -1, s["k_cache"].shape[0]
    agrees(s, tree(2, 3))
    with pytest.raises(RuntimeError, match="outside the cache"):
        ops.check_status()
    k, v = ht.cache_gather(s["k_cache"], s["v_cache"], s["block_table"], s["lengths"], 100)
    for b, x in enumerate([100, 90]):
        assert torch.equal(k[b, :x].cpu(), oracle.cached_rows(s["k_cache"].cpu(), s["block_table"][b].cpu(), x)[0])
    with pytest.raises(RuntimeError, match="outside the cache"):
        ops.check_status()
    # lengths that no table row can name, or none at all: what there is
    t = make(dt, 3, 8, 2, 64, 64, 16, [32, 0], spare=2)
    t["block_table"] = t["block_table"][:, :2].contiguous()
    full = dict(t, lengths=_ints([32, 0]))
    want = ht.draft_attention(**full)
    assert torch.equal(ht.draft_attention(**dict(t, lengths=_ints([10 ** 9, -5]))), want)
    with pytest.raises(RuntimeError, match="outside the cache"):
        ops.check_status()
    # a draft whose parent comes after it continues the cached tokens
    par = _ints([[-1, 2, 0], [-1, -1, 2]])
    assert torch.equal(ht.draft_attention(**full, parents=par), ht.draft_attention(**full, parents=_ints([[-1, -1, 0], [-1, -1, -1]])))
    with pytest.raises(RuntimeError, match="outside the cache"):
        ops.check_status()


def test_empty_calls():
    import htree_b200 as ht
    s = make(BF, 2, 4, 2, 64, 64, 16, [20])
    z = {n: s[n][:, :0] if n in ("q", "k", "v") else s[n] for n in s}
    assert ht.draft_attention(**z).shape == (1, 0, 4, 64)
    z = {n: s[n] if n.endswith("cache") else s[n][:0] for n in s}
    assert ht.draft_attention(**z).shape == (0, 2, 4, 64)
    assert ht.cache_gather(s["k_cache"], s["v_cache"], s["block_table"], s["lengths"], 0)[0].shape == (1, 0, 2, 64)
    ht.cache_append(s["k"], s["v"], s["k_cache"], s["v_cache"], torch.empty(1, 0, dtype=torch.int64, device=DEV))
    all_pad = ht.draft_attention(**s, parents=_ints([[-2, -7]]), return_lse=True)
    assert (all_pad[0] == 0).all() and (all_pad[1] == -math.inf).all()


def test_refusals():
    import htree_b200 as ht
    s = make(BF, 3, 8, 2, 64, 64, 16, [40, 5])

    def no(match, exc=ValueError, **kw):
        with pytest.raises(exc, match=match):
            ht.draft_attention(**dict(s, **kw))

    no("q must be", q=s["q"].float())
    no("divisible", q=s["q"][:, :, :7])
    no("same row width", q=torch.zeros(2, 3, 8, 32, dtype=BF, device=DEV))
    no("same requests and drafts", q=s["q"][:, :2])
    no("heads and row widths", k=s["k"][:, :, :1])
    no("one row per request", lengths=s["lengths"][:1])
    no("lengths must be", lengths=s["lengths"].long())
    no("block_table must be", block_table=s["block_table"].long())
    no("parents must have one entry", parents=tree(2, 4))
    no("parents must be", parents=tree(2, 3).long())
    no("share one of", k_cache=s["k_cache"].double(), v_cache=s["v_cache"].double())
    no("same pages", v_cache=s["v_cache"][:-1])
    no("multiples of 8", k_cache=s["k_cache"][..., :60])
    no("dense", k_cache=s["k_cache"].transpose(1, 3).contiguous().transpose(1, 3))
    no("is on cpu", lengths=s["lengths"].cpu())
    no("CUDA", RuntimeError, k_cache=s["k_cache"].cpu())
    no("no backward", RuntimeError, q=s["q"].clone().requires_grad_())
    no("up to 1024", **{n: torch.zeros(2, 1025, s[n].shape[2], 64, dtype=BF, device=DEV) for n in "qkv"}, parents=tree(2, 1025))
    wide = make(BF, 1, 2, 1, 264, 264, 16, [4])
    with pytest.raises(ValueError, match="up to 256"):
        ht.draft_attention(**wide)
    with torch.no_grad():
        ht.draft_attention(**dict(s, q=s["q"].clone().requires_grad_()))
    slots = torch.zeros(2, 3, dtype=torch.int64, device=DEV)
    for kw, match in ((dict(slots=slots.int()), "slots must be"), (dict(slots=slots[:1]), "one row per request"),
                      (dict(slots=torch.zeros(2, 4, dtype=torch.int64, device=DEV)), "pass index"), (dict(index=_ints([[0, 0]] * 2)), "shape of slots"),
                      (dict(k_cache=s["k_cache"][:1].expand(5, -1, -1, -1), v_cache=s["v_cache"][:1].expand(5, -1, -1, -1)), "expanded")):
        with pytest.raises(ValueError, match=match):
            ht.cache_append(**dict(dict(k=s["k"], v=s["v"], k_cache=s["k_cache"], v_cache=s["v_cache"], slots=slots), **kw))
    lens, table, pool, top = _ints([0, 0]), _ints([[-1] * 4] * 2), _ints([0, 1, 2]), _ints([3])
    for args, match in (((lens, lens[:1], table, pool, top, 16, 4), "one entry per request"), ((lens, lens, table.t(), pool, top, 16, 4), "one row per request"),
                        ((lens, lens, table, pool, top, 0, 4), "page_size"), ((lens, lens, table, pool, top, 16, 0), "n must be positive"),
                        ((lens, lens, table, pool, _ints([1, 2]), 16, 4), "top must be"), ((lens, lens, table[:, ::2], pool, top, 16, 4), "dense")):
        with pytest.raises(ValueError, match=match):
            ht.cache_plan(*args)


@pytest.mark.parametrize("B,M,page,n,pages", [(1, 4, 16, 20, 5), (7, 9, 4, 30, 40), (33, 40, 1, 25, 500), (700, 30, 16, 64, 9000), (1300, 9, 4, 12, 7000), (3, 6000, 2, 11000, 9000),
                                              (40, 700, 16, 3000, 9000)])
def test_plan(B, M, page, n, pages):
    """Turns of a batch that grows, runs out of pages, ends and goes on."""
    import htree_b200 as ht
    from htree_b200 import ops
    rng = random.Random(B * M)
    lens, table, pool, top = [0] * B, [[-1] * M for _ in range(B)], rng.sample(range(pages), pages), pages
    dl, dt, dp, dtop = _ints(lens), _ints(table), _ints(pool), _ints([top])
    for turn in range(6):
        counts = [rng.choice([-1, 0, 1, rng.randint(1, n), n, n + 1 if turn == 4 else 2]) for _ in range(B)]
        if turn == 0:
            counts = [rng.randint(1, n) for _ in range(B)]
        refused = any(c > n or c > 0 and x + c > M * page for c, x in zip(counts, lens))
        slots, taken = ht.cache_plan(dl, _ints(counts), dt, dp, dtop, page, n)
        s, t, lens, table, pool, top = oracle.plan(lens, counts, table, pool, top, page, n)
        assert taken.tolist() == t and dl.tolist() == lens and dtop.tolist() == [top]
        assert dt.tolist() == table and dp.tolist()[:top] == pool[:top] and slots.tolist() == s
        if refused:
            with pytest.raises(RuntimeError, match="block table"):
                ops.check_status()
    held = [p for r in table for p in r if p >= 0] + pool[:top]
    assert sorted(held) == list(range(pages))                # every page has one owner


def test_plan_with_bad_state_stays_inside_its_buffers():
    import htree_b200 as ht
    from htree_b200 import ops
    table = torch.full((6, 5), -9, dtype=torch.int32, device=DEV)      # 4 columns are passed; a guard row and a guard column
    table[:5, :4] = _ints([[0, 1, 2, 3]] * 5)
    pool = torch.full((8,), -9, dtype=torch.int32, device=DEV)
    pool[:6] = _ints([4, 5, 6, 7, 8, 9])
    lens, top = _ints([1000, -3, 64, 64, 64]), _ints([50])
    ht.cache_plan(lens, _ints([-1, 5, -1, -1, -1]), table[:5, :4], pool[:6], top, 16, 8)
    with pytest.raises(RuntimeError, match="outside the cache"):
        ops.check_status()
    assert (table[5] == -9).all() and (table[:, 4] == -9).all() and (pool[6:] == -9).all()
    assert 0 <= int(top) <= 6 and lens.tolist()[0] == 0


@pytest.mark.parametrize("dt,Hkv,K,V,page", [(BF, 2, 128, 128, 16), (HF, 1, 8, 24, 3), (FP, 8, 128, 64, 64), (BF, 5, 80, 256, 1), (FP, 3, 256, 256, 7)])
def test_append_and_gather(dt, Hkv, K, V, page):
    import htree_b200 as ht
    from htree_b200 import ops
    g = torch.Generator(device=DEV).manual_seed(K)
    B, N, n, P = 5, 23, 11, 200 // page + 60
    k, v = (torch.randn(B, N, Hkv, w, generator=g, device=DEV).to(dt) for w in (K, V))
    kc, vc = (torch.full((P, page, Hkv, w), 7.0, dtype=dt, device=DEV) for w in (K, V))
    lens, table = _ints([0] * B), torch.full((B, 40), -1, dtype=torch.int32, device=DEV)
    pool, top = torch.randperm(P, device=DEV).int(), _ints([P])
    counts = [23, 1, 0, 9, 16]
    slots, _ = ht.cache_plan(lens, _ints(counts), table, pool, top, page, N)
    ht.cache_append(k, v, kc, vc, slots)
    index = _ints([[(3 * i + b) % N for i in range(n)] for b in range(B)])
    more = [2, 11, 0, 5, 0]
    slots2, _ = ht.cache_plan(lens, _ints(more), table, pool, top, page, n)
    ht.cache_append(k, v, kc, vc, slots2, index)
    gk, gv = ht.cache_gather(kc, vc, table, lens, 40)
    hk, hv = ht.cache_gather(kc, vc, table, lens, 9)
    held = set()
    for b in range(B):
        L = counts[b] + more[b]
        for x, got, short in ((k, gk, hk), (v, gv, hv)):
            want = torch.cat([x[b, :counts[b]], x[b, index[b, :more[b]].long()]])
            assert torch.equal(got[b, :L], want) and (got[b, L:] == 0).all() and torch.equal(short[b], got[b, :9])
        held |= {int(table[b, i // page]) * page + i % page for i in range(L)}
    rest = torch.ones(P * page, dtype=torch.bool, device=DEV)
    rest[list(held)] = False
    assert (kc.view(-1, Hkv, K)[rest] == 7).all() and (vc.view(-1, Hkv, V)[rest] == 7).all()
    # slots and tokens that do not exist: not written, reported; strided sources and caches
    before = kc.clone()
    for sl, ix in ((P * page, 0), (-2, 0), (5, N), (5, -1)):
        ht.cache_append(k[:1], v[:1], kc, vc, torch.tensor([[sl]], device=DEV), _ints([[ix]]))
        with pytest.raises(RuntimeError, match="outside the cache"):
            ops.check_status()
    assert torch.equal(before, kc)
    kv = torch.cat([k, v], -1) if K == V else None
    if kv is not None:
        both = torch.zeros(P, Hkv, page, 2 * K, dtype=dt, device=DEV)
        ht.cache_append(kv[..., :K], kv[..., K:], both[..., :K].transpose(1, 2), both[..., K:].transpose(1, 2), slots)
        a, b = ht.cache_gather(both[..., :K].transpose(1, 2), both[..., K:].transpose(1, 2), table, _ints(counts), N)
        for i in range(B):
            assert torch.equal(a[i, :counts[i]], k[i, :counts[i]]) and torch.equal(b[i, :counts[i]], v[i, :counts[i]])


def test_what_is_written_is_known_to_autograd():
    """A tensor saved for a backward pass and written since is an error there, not a wrong gradient."""
    import htree_b200 as ht
    kc, vc = torch.ones(4, 8, 1, 16, device=DEV), torch.ones(4, 8, 1, 16, device=DEV)
    k = torch.zeros(1, 1, 1, 16, device=DEV)
    w = torch.ones(16, device=DEV, requires_grad=True)
    loss = (w * kc).sum()
    ht.cache_append(k, k, kc, vc, torch.zeros(1, 1, dtype=torch.int64, device=DEV))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    lengths, table, pool, top = _ints([0]), _ints([[-1, -1]]), _ints([0, 1]), _ints([2])
    before = [x._version for x in (lengths, table, pool, top)]
    ht.cache_plan(lengths, _ints([3]), table, pool, top, 8, 3)
    assert all(x._version > n for x, n in zip((lengths, table, pool, top), before))
    with torch.inference_mode():
        kc = torch.ones(4, 8, 1, 16, device=DEV)
        ht.cache_append(k, k, kc, kc.clone(), torch.zeros(1, 1, dtype=torch.int64, device=DEV))
    ht.cache_append(k, k, kc, torch.ones_like(kc), torch.ones(1, 1, dtype=torch.int64, device=DEV))
    assert kc[0, :2].abs().sum() == 0


def test_parts_join_by_their_lse():
    """Attention over two halves of 320 tokens (the last of each as the draft), joined by lse, is attention over the whole."""
    import htree_b200 as ht
    s = make(FP, 1, 8, 2, 64, 64, 16, [320])
    token = lambda i: {n: s[n + "_cache"][s["block_table"][0, i // 16].long(), i % 16].view(1, 1, 2, 64) for n in "kv"}      # noqa: E731
    part = lambda at, n: ht.draft_attention(**dict(s, block_table=s["block_table"][:, at // 16:].contiguous(), lengths=_ints([n - 1]),      # noqa: E731
                                                   **token(at + n - 1)), return_lse=True)
    whole, lse = part(0, 320)
    first, rest = part(0, 160), part(160, 160)
    w = torch.softmax(torch.stack([first[1], rest[1]]), 0)
    # by the oracle's count a part is good to 5e-5 of values around 1 (scores of 64 products of sum 5: 2e-5, twice; n * 2^-23)
    assert (w[0, ..., None] * first[0] + w[1, ..., None] * rest[0] - whole).abs().max() < 2e-4
    assert (torch.logsumexp(torch.stack([first[1], rest[1]]), 0) - lse).abs().max() < 1e-4


def test_generation():
    """The calls as a program makes them: prompts in, turns of drafted trees of which a path is accepted, requests that end and begin;
    attention against the oracle over what was accepted, the cache against a list of it, and htree_forward on the gathered cache."""
    import htree_b200 as ht
    g = torch.Generator(device=DEV).manual_seed(9)
    rng = random.Random(9)
    B, H, Hkv, D, page, P, N = 4, 8, 2, 64, 16, 80, 6
    kc, vc = (torch.full((P, page, Hkv, D), math.nan, dtype=BF, device=DEV) for _ in range(2))
    lens, table = _ints([0] * B), torch.full((B, 24), -1, dtype=torch.int32, device=DEV)
    pool, top = torch.arange(P, device=DEV, dtype=torch.int32), _ints([P])
    held = [[] for _ in range(B)]
    new = lambda n: [torch.randn(B, n, h, D, generator=g, device=DEV).to(BF) for h in (H, Hkv, Hkv)]      # noqa: E731
    prompt = [100, 33, 1, 64]
    q, k, v = new(100)
    chunk = agrees(dict(q=q[:, :40], k=k[:, :40], v=v[:, :40], k_cache=kc, v_cache=vc, block_table=table, lengths=lens))
    assert torch.isfinite(chunk[0]).all()
    slots, taken = ht.cache_plan(lens, _ints(prompt), table, pool, top, page, 100)
    assert taken.tolist() == prompt
    ht.cache_append(k, v, kc, vc, slots)
    for b in range(B):
        held[b] = [(k[b, i], v[b, i]) for i in range(prompt[b])]
    for turn in range(5):
        q, k, v = new(N)
        par = tree(B, N, seed=turn)
        agrees(dict(q=q, k=k, v=v, k_cache=kc, v_cache=vc, block_table=table, lengths=lens), par)
        paths = []
        for b in range(B):
            leaf, path = rng.randrange(N), []
            while leaf >= 0:
                path.insert(0, leaf)
                leaf = int(par[b, leaf])
            paths.append(path)
        counts = [len(p) if not (turn == 2 and b == 1) else -1 for b, p in enumerate(paths)]
        slots, taken = ht.cache_plan(lens, _ints(counts), table, pool, top, page, N)
        ht.cache_append(k, v, kc, vc, slots, _ints([p + [0] * (N - len(p)) for p in paths]))
        for b in range(B):
            held[b] = [] if counts[b] < 0 else held[b] + [(k[b, i], v[b, i]) for i in paths[b]]
        assert lens.tolist() == [len(x) for x in held]
    T = max(len(x) for x in held)
    gk, gv = ht.cache_gather(kc, vc, table, lens, T)
    dense = [torch.zeros(B, T, Hkv, D, dtype=BF, device=DEV) for _ in range(2)]
    for b in range(B):
        for i, (a, c) in enumerate(held[b]):
            dense[0][b, i], dense[1][b, i] = a, c
    assert torch.equal(gk, dense[0]) and torch.equal(gv, dense[1])
    b = max(range(B), key=lambda x: len(held[x]))
    args = dict(compression_rate=16, max_top_nodes=64, top_k_per_layer=16)
    a, c = (ht.htree_forward(q[b:b + 1, -1:], x[b:b + 1], y[b:b + 1], _q_offset=T - 1, **args) for x, y in ((gk, gv), dense))
    assert torch.equal(a, c) and torch.isfinite(a).all()


@pytest.mark.parametrize("dt", [FP, BF])
def test_streams_and_graphs(dt):
    """Other streams at the same time, and turns captured once and replayed on changed contents, two graphs in turn."""
    import htree_b200 as ht
    s1, s2 = make(dt, 4, 8, 2, 64, 64, 16, [700, 90], seed=1), make(dt, 7, 8, 2, 64, 64, 16, [3000, 4], seed=2)
    p1, p2 = tree(2, 4), tree(2, 7)
    want1, want2 = ht.draft_attention(**s1, parents=p1), ht.draft_attention(**s2, parents=p2)
    torch.cuda.synchronize()
    st = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [[], []]
    for _ in range(20):
        for i, (s, p) in enumerate(((s1, p1), (s2, p2))):
            with torch.cuda.stream(st[i]):
                outs[i].append(ht.draft_attention(**s, parents=p))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want1) for x in outs[0]) and all(torch.equal(x, want2) for x in outs[1])

    P, page = 60, 16
    kc, vc = (torch.zeros(P, page, 2, 64, dtype=dt, device=DEV) for _ in range(2))
    lens, table, pool, top = _ints([0, 0]), torch.full((2, 20), -1, dtype=torch.int32, device=DEV), torch.arange(P, device=DEV, dtype=torch.int32), _ints([P])
    counts, index = _ints([3, 0]), _ints([[0, 1, 3, 0], [2, 0, 0, 0]])
    q, k, v = (s1[n].clone() for n in "qkv")

    def turn():
        out = ht.draft_attention(q, k, v, kc, vc, table, lens, p1)
        slots, _ = ht.cache_plan(lens, counts, table, pool, top, page, 4)
        ht.cache_append(k, v, kc, vc, slots, index)
        return out

    graphs, got = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            got.append(turn())
        graphs.append(gr)
    kc2, vc2, lens2, table2, pool2, top2 = (x.clone() for x in (kc, vc, lens, table, pool, top))
    for i in range(8):
        k.copy_(torch.randn_like(k)); v.copy_(torch.randn_like(v)); q.copy_(torch.randn_like(q))
        counts.copy_(_ints([1 + i % 3, (i % 2) * 4]))
        graphs[i % 2].replay()
        out = ht.draft_attention(q, k, v, kc2, vc2, table2, lens2, p1)
        slots, _ = ht.cache_plan(lens2, counts, table2, pool2, top2, page, 4)
        ht.cache_append(k, v, kc2, vc2, slots, index)
        assert torch.equal(got[i % 2], out)
    for a, b in ((kc, kc2), (vc, vc2), (lens, lens2), (table, table2), (pool, pool2), (top, top2)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dt", [FP, BF, HF])
def test_calls_repeat_bit_for_bit(dt):
    import htree_b200 as ht
    s = make(dt, 5, 16, 2, 128, 128, 16, [5000, 1, 800])
    first = ht.draft_attention(**s, parents=tree(3, 5), return_lse=True)
    for _ in range(5):
        for a, b in zip(first, ht.draft_attention(**s, parents=tree(3, 5), return_lse=True)):
            assert torch.equal(a, b)


# Heights, in units of the exponent, around what fp32 holds of a power of two (2^128 is e^88.7), of one with a sign (2^256, 2^384: e^177, e^266) and far beyond.
HEIGHTS = [60, 86, 88, 89, 90, 92, 100, 110, 150, 176, 178, 220, 265, 267, 300, 350, 400, 600]


def steep(dt, N, G, K, lengths, seed=0):
    """One height for all rows of a request and key/value head (rows of a warp would otherwise look for the maximum together): their scores over a
    key along a common direction (8 in every element) are that, over other keys next to nothing.  Returns the state and the direction."""
    s = make(dt, N, 2 * G, 2, K, K, 16, lengths, seed=seed)
    height = torch.tensor([[HEIGHTS[(5 * b + 9 * h + seed) % len(HEIGHTS)] for h in range(2)] for b in range(len(lengths))], device=DEV, dtype=torch.float32)
    s["q"] = (0.1 * s["q"].float() + (height / (8 * K ** 0.5)).repeat_interleave(G, 1)[:, None, :, None]).to(dt)
    for n in ("k", "k_cache"):
        s[n] = (s[n].float() - s[n].float().mean(-1, keepdim=True)).to(dt)
    return s, torch.full((K,), 8.0, device=DEV)


def at_token(s, b, pos):
    return s["block_table"][b, pos // 16].long(), pos % 16


@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("N,G,K", [(20, 2, 64), (40, 4, 64), (20, 2, 128), (40, 4, 128), (6, 2, 128)])
@pytest.mark.parametrize("first", [0, 49, 210])
def test_one_key_far_above_the_others(dt, N, G, K, first):
    """At every place of sixteen, among the first tokens, later ones and those of a later tile, few to very many units above the rest."""
    s, far = steep(dt, N, G, K, [300] * 16, seed=first)
    for b in range(16):
        page, place = at_token(s, b, first + b)
        s["k_cache"][page, place] = far.to(dt)
    agrees(s, tree(16, N, seed=first))


@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("N,G,K", [(20, 2, 64), (40, 4, 128)])
def test_first_keys_far_below_the_others(dt, N, G, K):
    """The first sixteen tokens, a whole tile of 128 or nearly all of them, and the drafts, far below what follows."""
    lengths = [300, 290, 400, 144, 17, 256, 512, 513]
    s, far = steep(dt, N, G, K, lengths, seed=1)
    for b, from_ in enumerate([16, 128, 256, 127, 16, 100, 255, 511]):
        for pos in range(from_, lengths[b]):
            page, place = at_token(s, b, pos)
            s["k_cache"][page, place] += far.to(dt)
    agrees(s, tree(8, N, seed=2))
    s["k"][:, 1::3] += far.to(dt)
    agrees(s)


@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("N,G,K", [(20, 2, 64), (40, 4, 128), (3, 2, 64)])
@pytest.mark.parametrize("first", [0, 49, 210])
def test_a_cached_key_that_is_nan_is_seen(dt, N, G, K, first):
    """At every place of sixteen: the rows of its request and head are NaN, and no others."""
    import htree_b200 as ht
    s = make(dt, N, 2 * G, 2, K, K, 16, [300] * 17)
    for b in range(16):
        page, place = at_token(s, b, first + b)
        s["k_cache"][page, place, b % 2, 3] = math.nan
    out, lse = ht.draft_attention(**s, return_lse=True)
    hit = torch.tensor([[b % 2 == h and b < 16 for h in range(2)] for b in range(17)], device=DEV).repeat_interleave(G, 1)[:, None].expand(17, N, 2 * G)
    assert out[hit].isnan().all() and lse[hit].isnan().all() and torch.isfinite(out[~hit]).all() and torch.isfinite(lse[~hit]).all()


def _of_no_page():
    """A call that reports a page outside the cache."""
    s = make(BF, 2, 4, 2, 64, 64, 16, [20])
    return dict(s, block_table=torch.full_like(s["block_table"], -1))


@pytest.fixture
def no_status_word(monkeypatch):
    """As on a device whose first call is still to come."""
    from htree_b200 import ops
    monkeypatch.delitem(ops._status_words, torch.device("cuda", torch.cuda.current_device()), raising=False)


def test_reports_of_a_first_call_in_inference_mode(no_status_word):
    import htree_b200 as ht
    from htree_b200 import ops
    with torch.inference_mode():
        ht.draft_attention(**_of_no_page())
    with pytest.raises(RuntimeError, match="outside the cache"):
        ops.check_status()
    ops.check_status()


def test_reports_of_a_first_call_in_a_capture(no_status_word):
    """The word that collects reports is not the graph's: a replay neither makes it nor clears it."""
    import htree_b200 as ht
    from htree_b200 import ops
    good, bad = make(BF, 2, 4, 2, 64, 64, 16, [20]), _of_no_page()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ht.draft_attention(**good)
    ops.check_status()
    ht.draft_attention(**bad)
    graph.replay()
    with pytest.raises(RuntimeError, match="outside the cache"):
        ops.check_status()
    assert torch.equal(out, ht.draft_attention(**good))


def test_tangents_are_refused():
    """No call has a forward-mode derivative either; without a tangent, or where tangents are off, they run."""
    import htree_b200 as ht
    import torch.autograd.forward_ad as fw
    s = make(BF, 2, 4, 2, 64, 64, 16, [20])
    slots = torch.zeros(1, 2, dtype=torch.int64, device=DEV)
    calls = {"q": ht.draft_attention, "k": ht.draft_attention, "v": ht.draft_attention, "k_cache": ht.draft_attention, "v_cache": ht.draft_attention}
    append = lambda **t: ht.cache_append(t["k"], t["v"], t["k_cache"], t["v_cache"], slots)      # noqa: E731
    gather = lambda **t: ht.cache_gather(t["k_cache"], t["v_cache"], t["block_table"], t["lengths"], 20)      # noqa: E731
    want = ht.draft_attention(**s)
    with fw.dual_level():
        for name in calls:
            t = dict(s, **{name: fw.make_dual(s[name], torch.ones_like(s[name]))})
            for call in [ht.draft_attention] + [append] * (name != "q") + [gather] * name.endswith("cache"):
                for grad in (torch.enable_grad, torch.no_grad):           # (no_grad leaves tangents on)
                    with grad(), pytest.raises(RuntimeError, match="no forward-mode derivative"):
                        call(**t)
            with fw._set_fwd_grad_enabled(False):
                assert torch.equal(ht.draft_attention(**t), want)
        assert torch.equal(ht.draft_attention(**s), want)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda q: ht.draft_attention(**dict(s, q=q)), (s["q"],), (torch.ones_like(s["q"]),))


@pytest.mark.parametrize("n,extra", [(64, 0), (20000, 0), (64, 1100)])
def test_plan_reports_pages_that_are_none(n, extra):
    """A length of more pages than the table row has: the entry goes round (a page for a page), but is reported when it is given back and when
    it is taken, and its tokens have no slots.  Slots by the plan itself and by the chip, few rows and more than a thousand."""
    import htree_b200 as ht
    from htree_b200 import ops
    B = 2 + extra
    lens, table = _ints([40, 0] + [0] * extra), _ints([[3, -1, 5, -1], [-1] * 4] + [[-1] * 4] * extra)
    pool, top = _ints([0, 1, 2, 9, 9, 9]), _ints([3])
    ht.cache_plan(lens, _ints([-1] + [0] * (B - 1)), table, pool, top, 16, n)
    with pytest.raises(RuntimeError, match="outside the cache"):
        ops.check_status()
    assert lens[:2].tolist() == [0, 0] and (table == -1).all() and pool.tolist() == [0, 1, 2, 3, -1, 5] and int(top) == 6
    slots, taken = ht.cache_plan(lens, _ints([0, 60] + [0] * extra), table, pool, top, 16, n)
    with pytest.raises(RuntimeError, match="outside the cache"):
        ops.check_status()
    assert taken[:2].tolist() == [0, 60] and table[1].tolist() == [5, -1, 3, 2]
    assert slots[1, :60].tolist() == list(range(80, 96)) + [-1] * 16 + list(range(48, 64)) + list(range(32, 44))
    assert (slots[1, 60:] == -1).all() and (slots[0] == -1).all() and (slots[2:] == -1).all()


# What the smaller tests ask of few query rows, of 40 to 160 (tcgen05 in 16 bits, tiles of 64 rows in fp32) and of wide ones.
MANY = [(BF, 40, 4, 128, 16), (HF, 20, 2, 64, 64), (BF, 20, 2, 128, 128), (HF, 40, 4, 64, 48), (BF, 40, 4, 128, 7), (BF, 20, 3, 64, 256), (FP, 20, 2, 64, 16),
        (FP, 40, 4, 128, 64), (BF, 40, 2, 256, 16)]


@pytest.mark.parametrize("dt,N,G,K,page", MANY)
def test_pages_outside_the_cache_with_many_rows(dt, N, G, K, page):
    """Bad pages among good ones, first and last ones, all of a request; lengths beyond the table; a draft before its parent."""
    import htree_b200 as ht
    from htree_b200 import ops
    s = make(dt, N, 2 * G, 2, K, K, page, [700, 520, 300, 129], seed=page)
    P, bad = s["k_cache"].shape[0], [-1, 2 ** 31 - 1, -2 ** 31]
    held = [-(-x // page) for x in (700, 520, 300, 129)]
    for b, at in enumerate([[0, held[0] // 2], [held[1] // 3, held[1] - 1], range(held[2]), [0]]):
        for i, j in enumerate(at):
            s["block_table"][b, j] = ([P] + bad)[(b + i) % 4]
    agrees(s, tree(4, N, pad=0.1))
    with pytest.raises(RuntimeError, match="outside the cache"):
        ops.check_status()
    t = make(dt, N, 2 * G, 2, K, K, page, [page * 3, 0], spare=2)
    t["block_table"] = t["block_table"][:, :3].contiguous()
    want = ht.draft_attention(**t)
    assert torch.equal(ht.draft_attention(**dict(t, lengths=_ints([2 ** 31 - 1, -5]))), want)
    with pytest.raises(RuntimeError, match="outside the cache"):
        ops.check_status()
    par = tree(2, N, seed=3)
    same, par[0, 1], par[1, 7] = par.clone(), 1, N + 5
    same[0, 1] = same[1, 7] = -1
    assert torch.equal(ht.draft_attention(**t, parents=par), ht.draft_attention(**t, parents=same))
    with pytest.raises(RuntimeError, match="outside the cache"):
        ops.check_status()


@pytest.mark.parametrize("dt,N,G,K", [(BF, 40, 4, 128), (HF, 20, 2, 64), (FP, 40, 1, 128)])
def test_offsets_beyond_32_bits_with_many_rows(dt, N, G, K):
    import htree_b200 as ht
    page, pages = 256, (9 << 28) // (256 * K)                            # 2.4e9 elements
    small = make(dt, N, G, 1, K, K, page, [1000])
    kc, vc = (torch.zeros(pages, page, 1, K, dtype=dt, device=DEV) for _ in range(2))
    used, far = small["block_table"][0, :4].long(), torch.arange(pages - 4, pages, device=DEV)
    kc[far], vc[far] = small["k_cache"][used], small["v_cache"][used]
    table = small["block_table"].clone()
    table[0, :4] = far.int()
    par = tree(1, N)
    assert torch.equal(ht.draft_attention(**dict(small, k_cache=kc, v_cache=vc, block_table=table), parents=par), ht.draft_attention(**small, parents=par))


@pytest.mark.parametrize("dt,K", [(BF, 128), (HF, 64), (FP, 128)])
def test_streams_graphs_and_repeats_with_many_rows(dt, K):
    import htree_b200 as ht
    s = [make(dt, 40, 8, 2, K, K, 16, [1700, 90, 0], seed=1), make(dt, 20, 4, 2, K, K, 64, [3000, 4], seed=2)]
    p = [tree(3, 40), tree(2, 20)]
    want = [ht.draft_attention(**x, parents=y, return_lse=True) for x, y in zip(s, p)]
    torch.cuda.synchronize()
    st, outs = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(st[i]):
                outs[i].append(ht.draft_attention(**s[i], parents=p[i], return_lse=True))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for got in outs[i] for a, b in zip(got, want[i]))
    graphs, got = [], []
    for i in (0, 1, 0):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            got.append(ht.draft_attention(**s[i], parents=p[i]))
    for turn in range(4):
        for x in s:
            for n in "qkv":
                x[n].copy_(torch.randn_like(x[n]))
            x["lengths"] -= 3 * (x["lengths"] > 50).int()
        for g in graphs:
            g.replay()
        for i, out in zip((0, 1, 0), got):
            assert torch.equal(out, ht.draft_attention(**s[i], parents=p[i]))


@pytest.mark.parametrize("dt,K", [(BF, 128), (HF, 64), (FP, 128), (BF, 256)])
def test_expanded_caches(dt, K):
    """Heads that share a row of the cache and requests that share drafts, read through strides of zero."""
    import htree_b200 as ht
    s = make(dt, 40, 8, 2, K, K, 16, [300, 64])
    e = dict(s, k_cache=s["k_cache"][:, :, :1].expand(-1, -1, 2, -1), v_cache=s["v_cache"][:, :, :1].expand(-1, -1, 2, -1), k=s["k"][:1].expand(2, -1, -1, -1),
             q=s["q"][:, :, :1].expand(-1, -1, 8, -1))
    for N in (40, 1):
        for n in "qkv":
            e[n] = e[n][:, :N]
        f = {n: x.contiguous() for n, x in e.items()}
        for a, b in zip(ht.draft_attention(**e, return_lse=True), ht.draft_attention(**f, return_lse=True)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dt,scale", [(FP, -0.7), (FP, 0.0), (BF, -1.0), (HF, 0.0), (BF, 3.0)])
def test_scales_with_many_rows(dt, scale):
    agrees(make(dt, 40, 8, 2, 128, 128, 16, [150, 300, 0]), tree(3, 40, pad=0.1), scale)


@pytest.mark.parametrize("dt,N,K,lengths,is_tree", [(BF, 2500, 128, [300], False), (FP, 1500, 64, [70], False), (HF, 1024, 64, [200], True), (FP, 1024, 32, [5], True),
                                                    (BF, 700, 256, [100], False), (BF, 1024, 96, [0], True)])
def test_long_chains_and_large_trees(dt, N, K, lengths, is_tree):
    agrees(make(dt, N, 1, 1, K, K, 16, lengths), tree(1, N, pad=0.02) if is_tree else None)


@pytest.mark.parametrize("dt", [BF, HF])
def test_exponentials_on_the_fma_pipes(dt):
    """Scores that are exact, of which those at places 6, 7, 14 and 15 of every sixteen make the sum: the lse shows their exponentials."""
    s = make(dt, 40, 1, 1, 8, 8, 16, [128] * 64)
    s["q"].zero_(); s["k"].zero_(); s["k_cache"].zero_()
    s["q"][..., 0], s["k"][..., 0], s["k_cache"][..., 0] = 1.0, -1000.0, -1000.0
    for b, x in enumerate(torch.linspace(-3.0, 6.5, 64).tolist()):
        pages = s["block_table"][b, :8].long()
        s["k_cache"][pages[0], 0, 0, 0] = 0.0                         # the reference
        for place in (6, 7, 14, 15):
            s["k_cache"][pages, place, 0, 0] = x
    agrees(s, scale=1.0)


@pytest.mark.parametrize("dt,N,G,K,page", MANY + [(BF, 1, 4, 64, 16), (HF, 5, 2, 128, 16), (FP, 3, 2, 64, 16)])
def test_scores_of_minus_infinity(dt, N, G, K, page):
    """A row whose every score is -inf is an empty row; among others, such a key is one that weighs nothing."""
    import htree_b200 as ht
    s = make(dt, N, 2 * G, 2, K, K, page, [300, 300])
    s["q"][..., 0] = 8.0
    far = dict(s, k=s["k"].clone(), k_cache=s["k_cache"].clone())
    for x, low in ((s, -math.inf), (far, -1000.0)):
        mine = x["block_table"][0, :-(-300 // page)].long()
        x["k_cache"][mine, ..., 0], x["k"][0, ..., 0] = low, low
        x["k_cache"][x["block_table"][1, :-(-300 // page):2].long(), :, :, 0], x["k"][1, 1::2, :, 0] = low, low
    out, lse = ht.draft_attention(**s, return_lse=True)
    assert (out[0] == 0).all() and (lse[0] == -math.inf).all()
    want = ht.draft_attention(**far, return_lse=True)
    assert torch.equal(out[1], want[0][1]) and torch.equal(lse[1], want[1][1]) and torch.isfinite(lse[1]).all()
