"""The paged cache's operators without a GPU: the C interface rejects bad arguments before any launch, the Python one refuses what has no
implementation, and the plain forms that the GPU tests compare with agree with simpler statements of the same things."""
import ctypes

import pytest
import torch

from htree_b200 import _lib
from tests import cache_oracle as oracle

P = 4096      # a pointer that is aligned and never followed


def _cache(**kw):
    c = dict(k=P, v=P, k_page=4096, k_row=128, k_head=64, v_page=4096, v_row=128, v_head=64, pages=8, page_size=32, H_kv=2, K=64, V=64, dtype=1)
    c.update(kw)
    return _lib.HtreeCache(*[c[n] for n, _ in _lib.HtreeCache._fields_])


def _drafts(**kw):
    s = (ctypes.c_int64 * 3)(64 * 8, 64 * 8, 64)
    d = dict(q=P, k=P, v=P, q_stride=s, k_stride=s, v_stride=s, table=P, lengths=P, parents=None, out=P, lse=None, table_stride=8, B=2, N=4, H=8,
             M=8, scale=0.125)
    d.update(kw)
    return _lib.HtreeDrafts(*[d[n] for n, _ in _lib.HtreeDrafts._fields_])


def _attend(cache, drafts, ws=P, ws_bytes=1 << 40):
    return _lib.lib().htree_b200_draft_attention(ctypes.byref(cache), ctypes.byref(drafts), ws, ws_bytes, None, None)


def test_draft_attention_rejects_before_any_launch():
    odd = (ctypes.c_int64 * 3)(512, 512, 60)
    back = (ctypes.c_int64 * 3)(512, -512, 64)
    assert _lib.lib().htree_b200_draft_workspace(ctypes.byref(_cache()), ctypes.byref(_drafts())) > 0
    before = _lib.launch_count()
    assert _attend(_cache(k=None), _drafts()) == -1
    assert _attend(_cache(), _drafts(q=None)) == -1
    assert _attend(_cache(), _drafts(lengths=None)) == -1
    assert _attend(_cache(), _drafts(), ws=None) == -1
    assert _attend(_cache(), _drafts(H=7)) == -2
    assert _attend(_cache(), _drafts(N=0)) == -2
    assert _attend(_cache(), _drafts(table_stride=4)) == -2
    assert _attend(_cache(page_size=0), _drafts()) == -2
    assert _attend(_cache(dtype=5), _drafts()) == -3
    assert _attend(_cache(K=60), _drafts()) == -7
    assert _attend(_cache(k=P + 8), _drafts()) == -7
    assert _attend(_cache(v_row=100), _drafts()) == -7
    assert _attend(_cache(), _drafts(q_stride=odd)) == -7
    assert _attend(_cache(), _drafts(k_stride=back)) == -7
    assert _attend(_cache(K=264), _drafts()) == -8
    assert _attend(_cache(V=264), _drafts()) == -8
    assert _attend(_cache(), _drafts(N=1025, parents=P)) == -8
    assert _attend(_cache(), _drafts(M=64, table_stride=64), ws_bytes=64) == -11      # (tables of a few hundred tokens need no more than a word)
    need = _lib.lib().htree_b200_draft_workspace(ctypes.byref(_cache()), ctypes.byref(_drafts(M=64, table_stride=64)))
    assert need > 64 and _attend(_cache(), _drafts(M=64, table_stride=64), ws_bytes=need - 1) == -11
    assert _lib.launch_count() == before


def test_the_other_calls_reject_before_any_launch():
    lib, before = _lib.lib(), _lib.launch_count()
    s = (ctypes.c_int64 * 3)(512, 128, 64)

    def plan(B=2, M=8, page=16, n=4, lengths=P, stride=8, pool_size=9, slots=P):
        return lib.htree_b200_cache_plan(B, M, page, n, lengths, P, P, stride, P, pool_size, P, slots, P, None, None)

    assert [plan(B=0), plan(M=0), plan(page=0), plan(n=0), plan(stride=7), plan(pool_size=0)] == [-2] * 6
    assert [plan(lengths=None), plan(slots=None)] == [-1] * 2
    assert [plan(B=65536), plan(page=(1 << 20) + 1)] == [-8] * 2

    def append(cache=None, B=2, N=4, n=4, k=P, ks=s, index=None, slots=P):
        return lib.htree_b200_cache_append(ctypes.byref(cache or _cache()), B, N, n, k, ks, P, s, slots, index, None, None)

    assert [append(B=0), append(N=0), append(n=0), append(n=5)] == [-2] * 4
    assert [append(k=None), append(slots=None), append(_cache(v=None))] == [-1] * 3
    assert [append(k=P + 4), append(ks=(ctypes.c_int64 * 3)(512, 128, 63)), append(_cache(V=12))] == [-7] * 3

    def gather(cache=None, B=2, M=8, T=4, stride=8, k=P):
        return lib.htree_b200_cache_gather(ctypes.byref(cache or _cache()), B, M, T, P, stride, P, k, P, None, None)

    assert [gather(B=0), gather(M=0), gather(T=0), gather(stride=1), gather(_cache(pages=0))] == [-2] * 5
    assert [gather(k=None), gather(_cache(dtype=9)), gather(k=P + 2), gather(B=70000)] == [-1, -3, -7, -8]
    assert _lib.launch_count() == before


def test_python_calls_refuse_cpu_tensors():
    import htree_b200 as ht
    x, c = torch.zeros(1, 1, 2, 8), torch.zeros(2, 4, 2, 8)
    i = torch.zeros(1, dtype=torch.int32)
    t = torch.zeros(1, 2, dtype=torch.int32)
    for call in (lambda: ht.draft_attention(x, x, x, c, c, t, i), lambda: ht.cache_gather(c, c, t, i, 4),
                 lambda: ht.cache_append(x, x, c, c, torch.zeros(1, 1, dtype=torch.int64)), lambda: ht.cache_plan(i, i, t, i, i, 4, 1)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_quotients_by_multiplication():
    """Positions to pages, as the kernels form them: exact for every divisor up to 2^20 and every position below 2^31."""
    g = torch.Generator().manual_seed(1)
    for d in [1, 2, 3, 5, 7, 16, 24, 63, 64, 65, 100, 1000, 4097, 65535, 65536, 65537, (1 << 20) - 1, 1 << 20]:
        s = max(d - 1, 0).bit_length()
        mul = ((1 << (31 + s)) + d - 1) // d
        assert mul < 1 << 32
        some = torch.randint(0, 1 << 31, (200,), generator=g).tolist()
        top = (1 << 31) - 1
        for n in some + [x // d * d for x in some] + [x // d * d - 1 for x in some if x >= d] + [0, 1, d - 1, d, top, top // d * d, top // d * d - 1]:
            assert (n * mul) >> (31 + s) == n // d, (n, d)


def test_plain_forms():
    m = oracle.sees([-1, 0, 0, 1, -2, -1], 6)
    assert [r.nonzero().flatten().tolist() for r in m] == [[0], [0, 1], [0, 2], [0, 1, 3], [], [5]]
    assert torch.equal(oracle.sees(None, 5), torch.ones(5, 5).tril().bool())
    # 3 pages of 4: two rows, the first served, the second out of pages; then the first ends and the second is served from its pages
    s, taken, lens, table, pool, top = oracle.plan([0, 0], [9, 2], [[-1] * 4, [-1] * 4], [7, 8, 9], 3, 4, 9)
    assert taken == [9, 0] and lens == [9, 0] and table[0] == [9, 8, 7, -1] and top == 0 and s[0] == [36, 37, 38, 39, 32, 33, 34, 35, 28]
    s, taken, lens, table, pool, top = oracle.plan(lens, [-1, 2], table, pool, top, 4, 9)
    assert taken == [0, 2] and lens == [0, 2] and table == [[-1] * 4, [7, -1, -1, -1]] and top == 2 and pool[:2] == [9, 8]
    # a chain over an empty cache is causal attention
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(1, 5, 2, 8, generator=g) for _ in range(3))
    out, lse, tol, _ = oracle.attention(q, k, v, torch.zeros(1, 4, 2, 8), torch.zeros(1, 4, 2, 8), torch.zeros(1, 1, dtype=torch.int32),
                                        torch.zeros(1, dtype=torch.int32))
    s = torch.einsum("bihd,bjhd->bhij", q.double(), k.double()) * 8 ** -0.5
    w = s.masked_fill(~torch.ones(5, 5).tril().bool(), float("-inf")).softmax(-1)
    assert torch.allclose(out, torch.einsum("bhij,bjhd->bihd", w, v.double()), atol=1e-12) and (tol < 1e-4).all()


def test_a_wait_that_ran_out_is_told_as_what_it_is(monkeypatch):
    """The pipelined forward leaves outputs unwritten, the attention over the cache goes on with what there is: nobody is told that wrong numbers are old ones."""
    from htree_b200 import ops
    word = torch.tensor([16], dtype=torch.int32)
    monkeypatch.setitem(ops._status_words, torch.device("cpu"), word)
    with pytest.raises(RuntimeError, match="0x10: .*bounded wait .*forward were not written, those of draft_attention are wrong"):
        ops.check_status("cpu")
    assert word.item() == 0
    ops.check_status("cpu")
