"""The operators around drafted tokens on the CPU: the oracle against closed forms, and what the entry points refuse."""
import ctypes
import math

import pytest
import torch


@pytest.fixture(scope="module")
def D():
    from oracle import drafts_oracle
    return drafts_oracle


# --------------------------------------------------------------------------------------------------------------- oracle
@pytest.mark.parametrize("probs", [False, True])
def test_verified_tokens_are_the_targets(D, probs):
    """Two tokens behind the last one, drawn from q or looked up, then whatever comes next: over a fine grid of random
    numbers the first token that comes out has the target's distribution exactly (to the grid)."""
    V, grid = 4, 14
    logits = torch.tensor([[0.3, -1.0, 1.2, 0.1]]).repeat(3, 1)
    p = torch.softmax(logits[0].double(), 0)
    q = torch.tensor([0.5, 0.25, 0.125, 0.125]).double()
    got = torch.zeros(V, dtype=torch.float64)
    u = [(i + 0.5) / grid for i in range(grid)]
    for x in range(V):
        for y in range(V):
            if probs:
                share = float(q[x] * q[y])
            else:
                share = 1.0 if (x, y) == (2, 0) else 0.0
            if share == 0.0:
                continue
            for a in u:
                for b in u:
                    for c in u:
                        path, _, nxt, _ = D.verify(logits, [0, x, y], [0, 3], [c, a, b], [-1, 0, 0],
                                                   q.repeat(3, 1) if probs else None, None)
                        first = [nxt[0], x, y][path[1]] if path[1] > 0 else nxt[0]
                        got[first] += share / grid ** 3
    # three numbers on a grid: each border falls at most half a step wrong, in each of three stages
    assert bool(((got - p).abs() < 1.5 / grid).all()), (got, p)


def test_verify_oracle_closed_forms(D):
    logits = torch.tensor([[0.0, 0.0], [0.0, -math.inf], [math.nan, 0.0], [-math.inf, -math.inf]])
    # p = (1/2, 1/2): token 1 passes below 1/2
    assert D.verify(logits[:1].repeat(2, 1), [0, 1], [0, 2], [0.7, 0.49], None, None, None)[:3] == ([0, 1], [2], [1])
    assert D.verify(logits[:1].repeat(2, 1), [0, 1], [0, 2], [0.7, 0.5], None, None, None)[:3] == ([0, -1], [1], [0])
    # greedy: ties to the first
    assert D.verify(logits[:1].repeat(2, 1), [0, 0], [0, 2], [0.7, 0.99], None, None, [0.0])[:3] == ([0, 1], [2], [0])
    # a distribution that is not there stops the path
    assert D.verify(logits[[0, 2]], [0, 1], [0, 2], [0.1, 0.1], None, None, None)[:3] == ([0, 1], [2], [-1])
    assert D.verify(logits[[3]], [0], [0, 1], [0.1], None, None, None)[:3] == ([0], [1], [-1])
    # q = p: always accepted; nothing left of p: drawn from p
    assert D.verify(logits[:1].repeat(2, 1), [0, 1], [0, 2], [0.7, 0.999], None, torch.full((2, 2), 0.5), None)[1] == [2]
    assert D.verify(logits[:1].repeat(2, 1), [0, 1], [0, 2], [0.7, 1.0], None, torch.full((2, 2), 0.5), None)[:3] == (
        [0, -1], [1], [1])


def test_tree_oracle_is_the_recurrence(D):
    """A line of tokens is the sequence of the recurrence's own oracle; two branches are two sequences."""
    from oracle import cores_oracle as C
    g = torch.Generator().manual_seed(1)
    n, HV = 5, 2
    q, k = (torch.randn(n, 128, generator=g).bfloat16() * 0.1 for _ in range(2))
    v, gate = torch.randn(n, HV * 128, generator=g).bfloat16(), -torch.rand(n, HV, generator=g)
    beta = torch.rand(n, HV, generator=g).bfloat16()
    state = torch.randn(1, HV, 128, 128, generator=g)
    o = D.linattn_tree(q, k, v, gate, beta, state, [0], [0, n], None, 0.3)[0]
    want, last = C.linattn(q, k, v, gate, beta, [n], state, 0.3)[:2]
    assert torch.allclose(o, want, rtol=1e-12, atol=1e-14)
    got = D.linattn_keep(k, v, gate, beta, state, [0], [0, n], list(range(n)), [n])[0]
    assert torch.allclose(got, last, rtol=1e-12, atol=1e-14)
    fork = D.linattn_tree(q, k, v, gate, beta, state, [0], [0, n], [-1, 0, 0, 2, 1], 0.3)[0]
    for branch in ([0, 1, 4], [0, 2, 3]):
        part = [x[branch] for x in (q, k, v, gate, beta)]
        want = C.linattn(*part, [3], state, 0.3)[0]
        assert torch.allclose(fork[branch], want, rtol=1e-12, atol=1e-14)


def test_pages_oracle(D):
    table, refs, ctx = [[3, 1, -1], [-1] * 3, [-1] * 3], [0, 1, 0, 1, 0], [20, 0, 0]
    assert D.resize(table, refs, [-1, 17, 0], 16) == [0, 0, 0]
    assert table == [[3, 1, -1], [0, 2, -1], [-1] * 3] and refs == [1, 1, 1, 1, 0]
    assert D.fork(table, ctx, refs, [0, 0, 0], 16) == [(-1, -1), (1, 0), (1, 2)]
    assert table == [[3, 1, -1], [3, 0, -1], [3, 2, -1]] and refs == [1, 1, 1, 3, 0] and ctx == [20] * 3
    # two slots change places: the last pages are read before they are free again
    assert D.fork(table, ctx, refs, [1, 0, -1], 16) == [(0, 2), (1, 4), (-1, -1)]
    assert refs == [0, 0, 1, 2, 1] and ctx == [20, 20, 0]
    # no page left
    refs = [1, 1, 1, 2, 1]
    assert D.fork(table, ctx, refs, [0, 1, 0], 16)[2] == (2, -1) and ctx == [20, 20, 16] and table[2] == [3, -1, -1]


# ------------------------------------------------------------------------------------------------------------- refusals
@pytest.fixture()
def p():
    buf = ctypes.create_string_buffer(1 << 12)
    q = ctypes.c_void_p(ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 16)
    q.keep = buf
    return q


def test_verify_refusals(pkg, p):
    L = pkg._lib.lib()
    odd = ctypes.c_void_p(p.value + 1)

    def call(logits=p, kind=1, ldl=10, tokens=p, ptr=p, u=p, parents=p, probs=p, pkind=0, ldp=10, temp=p, N=3, B=2, V=10,
             path=p, count=p, nxt=p, ws=p, nws=1 << 20):
        return L.ojx_verify_drafts(logits, kind, ldl, tokens, ptr, u, parents, probs, pkind, ldp, temp, N, B, V, path, count,
                                   nxt, ws, nws, None)

    for bad in (dict(N=-1), dict(N=1 << 24), dict(B=-1), dict(B=65537), dict(V=0), dict(V=(1 << 22) + 1),
                dict(N=1 << 20, V=1 << 20, ldl=1 << 20, ldp=1 << 20)):
        assert call(**bad) == 2, bad
        assert L.ojx_verify_drafts_workspace(bad.get("N", 3), bad.get("B", 2), bad.get("V", 10), 1) == -1
    for bad in (dict(kind=2), dict(pkind=-1), dict(ldl=9), dict(ldp=9), dict(ldl=1 << 31), dict(logits=None), dict(tokens=None),
                dict(ptr=None), dict(u=None), dict(path=None), dict(count=None), dict(nxt=None), dict(logits=odd),
                dict(probs=odd), dict(tokens=ctypes.c_void_p(p.value + 4)), dict(u=odd), dict(temp=odd), dict(parents=odd)):
        assert call(**bad) == 1, bad
    for bad in (dict(ws=None), dict(nws=8), dict(ws=ctypes.c_void_p(p.value + 8))):
        assert call(**bad) == 3, bad
    assert call(N=0, B=0, logits=None, tokens=None, ptr=None, path=None) == 0
    assert 0 < L.ojx_verify_drafts_workspace(768, 64, 131072, 0) < L.ojx_verify_drafts_workspace(768, 64, 131072, 1)


def test_lintree_refusals(pkg, p):
    L = pkg._lib.lib()
    mis = ctypes.c_void_p(p.value + 2)

    def tree(q=p, k=p, g=p, beta=p, state=p, slot=p, slots=4, ptr=p, parents=p, N=3, B=2, HV=6, HK=2, o=p, ws=p, nws=1 << 30):
        return L.ojx_linattn_tree(q, k, p, g, beta, state, slot, slots, ptr, parents, N, B, HV, HK, 0.1, o, ws, nws, None)

    def keep(k=p, g=p, beta=p, state=p, slot=p, slots=4, ptr=p, path=p, count=p, N=3, B=2, HV=6, HK=2):
        return L.ojx_linattn_keep(k, p, g, beta, state, slot, slots, ptr, path, count, N, B, HV, HK, None)

    for bad in (dict(HK=0), dict(HK=4), dict(HV=2048, HK=2), dict(N=-1), dict(N=1 << 31), dict(B=-1), dict(slots=-1),
                dict(slots=1 << 31), dict(N=(1 << 24) // 6 + 1), dict(B=(1 << 24) // 6)):
        assert tree(**bad) == 2 and keep(**bad) == 2, bad
        if "slots" not in bad:
            assert L.ojx_linattn_tree_workspace(bad.get("N", 3), bad.get("B", 2), bad.get("HV", 6), bad.get("HK", 2)) == -1
    for bad in (dict(k=None), dict(g=None), dict(state=None), dict(slot=None), dict(ptr=None), dict(k=mis), dict(state=mis),
                dict(slot=mis), dict(ptr=mis), dict(g=mis)):
        assert tree(**bad) == 1 and keep(**bad) == 1, bad
    for bad in (dict(q=None), dict(o=None), dict(q=mis), dict(o=mis), dict(parents=mis)):
        assert tree(**bad) == 1, bad
    for bad in (dict(path=None), dict(count=None), dict(path=mis), dict(count=mis)):
        assert keep(**bad) == 1, bad
    for bad in (dict(ws=None), dict(nws=16), dict(ws=mis)):
        assert tree(N=65, **bad) == 3, bad            # longer sequences than a workgroup takes at once
    assert L.ojx_linattn_tree_workspace(64, 2, 6, 2) == 0 and L.ojx_linattn_tree_workspace(65, 2, 6, 2) == 65 * 6 * 552
    assert tree(N=0, k=None, q=None) == 0 and keep(N=0, k=None) == 0


def test_pages_refusals(pkg, p):
    L = pkg._lib.lib()
    mis = ctypes.c_void_p(p.value + 2)

    def resize(table=p, MP=4, refs=p, pages=8, tokens=p, B=2, page=16, out=p, ws=p, nws=1 << 20):
        return L.ojx_kv_pages_resize(table, MP, refs, pages, tokens, B, page, out, ws, nws, None)

    def fork(table=p, MP=4, refs=p, pages=8, tokens=p, B=2, page=16, out=p, ws=p, nws=1 << 20):
        return L.ojx_kv_pages_fork(table, MP, p, refs, pages, tokens, B, page, out, ws, nws, None)

    for f in (resize, fork):
        for bad in (dict(MP=-1), dict(MP=1 << 31), dict(B=-1), dict(B=65537), dict(B=65536, MP=1 << 15), dict(pages=-1),
                    dict(pages=1 << 31), dict(page=0), dict(page=24), dict(page=2048)):
            assert f(**bad) == 2, bad
        for bad in (dict(table=None), dict(refs=None), dict(tokens=None), dict(out=None), dict(table=mis), dict(refs=mis),
                    dict(tokens=mis), dict(out=mis)):
            assert f(**bad) == 1, bad
        for bad in (dict(ws=None), dict(nws=8), dict(ws=mis)):
            assert f(**bad) == 3, bad
        assert f(B=0, table=None, tokens=None) == 0
    for bad in ((-1, 4, 8), (65537, 4, 8), (2, -1, 8), (2, 1 << 31, 8), (65536, 1 << 15, 8), (2, 4, -1), (2, 4, 1 << 31)):
        assert L.ojx_kv_pages_workspace(*bad, 0) == -1 and L.ojx_kv_pages_workspace(*bad, 1) == -1

    def copy(kc=p, ks=p, fmt=1, layers=2, pages=8, HKV=2, page=16, D=256, pairs=p, n=3):
        return L.ojx_kv_pages_copy(kc, p, ks, p, fmt, layers, pages, HKV, page, D, pairs, n, None)

    def keep(kc=p, ks=p, fmt=1, layers=2, pages=8, HKV=2, page=16, D=256, table=p, MP=4, ctx=p, path=p, N=5, B=2):
        return L.ojx_kv_cache_keep(kc, p, ks, p, fmt, layers, pages, HKV, page, D, table, MP, ctx, p, path, p, N, B, None)

    for f in (copy, keep):
        for bad in (dict(layers=-1), dict(layers=65536), dict(layers=20000), dict(pages=-1), dict(pages=1 << 31), dict(HKV=0),
                    dict(HKV=1025), dict(page=8), dict(D=64)):
            assert f(**bad) == 2, bad
        for bad in (dict(fmt=2), dict(kc=None), dict(ks=None), dict(kc=mis), dict(ks=mis)):
            assert f(**bad) == 1, bad
        assert f(layers=0, kc=None) == 0
    assert copy(n=-1) == 2 and copy(n=65536) == 2 and copy(n=65535, layers=1000, page=1024) == 2
    assert copy(pairs=None) == 1 and copy(pairs=mis) == 1 and copy(n=0, pairs=None) == 0
    for bad in (dict(MP=-1), dict(N=-1), dict(B=-1), dict(B=65537), dict(B=65536, layers=100)):
        assert keep(**bad) == 2, bad
    for bad in (dict(table=None), dict(ctx=None), dict(path=None), dict(ctx=mis), dict(path=mis)):
        assert keep(**bad) == 1, bad
    assert keep(N=0, table=None) == 0


def test_python_refusals(ext):
    """CPU tensors are refused like everywhere in the package."""
    x, g = torch.zeros(3, 256, dtype=torch.bfloat16), torch.zeros(3, 2)
    kc = torch.zeros(4, 2, 16, 256, dtype=torch.bfloat16)
    i32, i64 = torch.zeros(3, dtype=torch.int32), torch.zeros(3, dtype=torch.int64)
    for call in (lambda: ext.linattn_tree(x, x, x, g, None, g, i32, i32), lambda: ext.linattn_keep(x, x, g, None, g, i32, i32, i32, i32),
                 lambda: ext.verify_drafts(x, i64, i32, g[:, 0]), lambda: ext.kv_cache_keep(kc, kc, i32, i32, i32, i32, i32),
                 lambda: ext.kv_pages_resize(i32[None], i32, i32, 16), lambda: ext.kv_pages_fork(i32[None], i32, i32, i32, 16),
                 lambda: ext.kv_pages_copy(kc, kc, i32)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_python_refusals_of_shapes(ext, monkeypatch):
    """Everything a kernel would read past is refused by its shape, before the library is called. (Tensors on the CPU pass
    the device checks here; the library must not be reached.)"""
    class Lib:
        def __getattr__(self, name):
            raise AssertionError(f"{name} was called")

    class Cuda(torch.Tensor):
        is_cuda = True

    monkeypatch.setattr(ext, "_chk", lambda t, name, dtype=None: None if t is not None and t.is_contiguous() and (
        dtype is None or t.dtype is dtype) else (_ for _ in ()).throw(RuntimeError(f"{name}")))
    monkeypatch.setattr(ext, "_one_device", lambda *a: None)
    monkeypatch.setattr(ext, "lib", Lib)
    z = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t).as_subclass(Cuda)  # noqa: E731
    f, i32, i64, e8 = torch.float32, torch.int32, torch.int64, torch.float8_e4m3fn
    x, tok, u, ptr = z(5, 30), z(5, t=i64), z(5, t=f), z(3, t=i32)
    for bad in (lambda: ext.verify_drafts(x.half(), tok, ptr, u), lambda: ext.verify_drafts(x[0], tok, ptr, u),
                lambda: ext.verify_drafts(x[:, :0], tok, ptr, u), lambda: ext.verify_drafts(x.T, z(30, t=i64), ptr, z(30, t=f)),
                lambda: ext.verify_drafts(x[:1].expand(5, 30), tok, ptr, u), lambda: ext.verify_drafts(x, tok[:4], ptr, u),
                lambda: ext.verify_drafts(x, tok.int(), ptr, u), lambda: ext.verify_drafts(x, tok, ptr.long(), u),
                lambda: ext.verify_drafts(x, tok, ptr[:0], u), lambda: ext.verify_drafts(x, tok, ptr, u[:4]),
                lambda: ext.verify_drafts(x, tok, ptr, u.double()), lambda: ext.verify_drafts(x, tok, ptr, u, ptr),
                lambda: ext.verify_drafts(x, tok, ptr, u, tok), lambda: ext.verify_drafts(x, tok, ptr, u, None, x[:4]),
                lambda: ext.verify_drafts(x, tok, ptr, u, None, x[:, :29]), lambda: ext.verify_drafts(x, tok, ptr, u, None, x.half()),
                lambda: ext.verify_drafts(x, tok, ptr, u, None, None, u), lambda: ext.verify_drafts(x, tok, ptr, u, None, None, ptr[:2]),
                lambda: ext.verify_drafts(x, None, ptr, u), lambda: ext.verify_drafts(x, tok, None, u)):
        with pytest.raises(RuntimeError):
            bad()
    y, v, g, b = z(5, 256), z(5, 768), z(5, 6, t=f), z(5, 6)
    st, slot, row = z(4, 6, 128, 128, t=f), z(2, t=i32), z(5, t=i32)
    ok = (y, y, v, g, b, st, slot, ptr)
    for bad in (lambda: ext.linattn_tree(y, z(5, 128), v, g, b, st, slot, ptr), lambda: ext.linattn_tree(y, y, z(4, 768), g, b, st, slot, ptr),
                lambda: ext.linattn_tree(y, y, v, g[:4], b, st, slot, ptr), lambda: ext.linattn_tree(y, y, v, g, b[:4], st, slot, ptr),
                lambda: ext.linattn_tree(y, y, v, g, b, st[:, :5], slot, ptr), lambda: ext.linattn_tree(y, y, v, g, b, st[0], slot, ptr),
                lambda: ext.linattn_tree(y, y, v, g, b, st, slot[:1], ptr), lambda: ext.linattn_tree(y, y, v, g, b, st, slot.long(), ptr),
                lambda: ext.linattn_tree(*ok[:7], ptr[:2]), lambda: ext.linattn_tree(*ok, row[:4]), lambda: ext.linattn_tree(*ok, row.long()),
                lambda: ext.linattn_tree(y, y, v, g, b, None, slot, ptr), lambda: ext.linattn_tree(y, y, v, g, b, st.bfloat16(), slot, ptr),
                lambda: ext.linattn_keep(*ok[1:], row[:4], slot), lambda: ext.linattn_keep(*ok[1:], row, slot[:1]),
                lambda: ext.linattn_keep(*ok[1:], None, slot), lambda: ext.linattn_keep(*ok[1:], row, None),
                lambda: ext.linattn_keep(*ok[1:], row.long(), slot), lambda: ext.linattn_keep(*ok[1:-1], ptr[:2], row, slot)):
        with pytest.raises(RuntimeError):
            bad()
    kc, k8, sc = z(4, 2, 16, 256), z(4, 2, 16, 256, t=torch.uint8).view(e8), z(4, 2, 16, t=f)
    k5, s5 = z(3, 4, 2, 16, 256, t=torch.uint8).view(e8), z(3, 4, 2, 16, t=f)
    table = z(2, 4, t=i32)
    rest = (table, slot, ptr, row, slot)
    for bad in (lambda: ext.kv_cache_keep(kc[0], kc[0], *rest), lambda: ext.kv_cache_keep(kc, kc[:3], *rest),
                lambda: ext.kv_cache_keep(k8, k8, *rest), lambda: ext.kv_cache_keep(k8, k8, *rest, sc, sc[:3]),
                lambda: ext.kv_cache_keep(kc, kc, *rest, sc, sc), lambda: ext.kv_cache_keep(k5, k5, *rest, s5, s5[:2]),
                lambda: ext.kv_cache_keep(k5, k5[0], *rest, s5, s5), lambda: ext.kv_cache_keep(k5, k5, *rest, sc, sc),
                lambda: ext.kv_cache_keep(kc, kc, table[:1], *rest[1:]), lambda: ext.kv_cache_keep(kc, kc, table.long(), *rest[1:]),
                lambda: ext.kv_cache_keep(kc, kc, table, slot[:1], *rest[2:]), lambda: ext.kv_cache_keep(kc, kc, table, slot, ptr, row, slot[:1]),
                lambda: ext.kv_cache_keep(kc, kc, table, slot, ptr, None, slot), lambda: ext.kv_cache_keep(kc, kc, table[0], *rest[1:]),
                lambda: ext.kv_pages_resize(table[0], row, slot, 16), lambda: ext.kv_pages_resize(table, row, slot[:1], 16),
                lambda: ext.kv_pages_resize(table, row.long(), slot, 16), lambda: ext.kv_pages_resize(table.long(), row, slot, 16),
                lambda: ext.kv_pages_fork(table, slot[:1], row, slot, 16), lambda: ext.kv_pages_fork(table, slot, row, slot[:1], 16),
                lambda: ext.kv_pages_fork(table, slot, row, slot.long(), 16), lambda: ext.kv_pages_copy(kc, kc, table),
                lambda: ext.kv_pages_copy(kc, kc, row), lambda: ext.kv_pages_copy(kc, kc, z(2, 2, t=i64)),
                lambda: ext.kv_pages_copy(k5, k5, z(2, 2, t=i32), s5)):
        with pytest.raises(RuntimeError):
            bad()


def test_verify_without_rows_has_no_walks(pkg):
    """Walks and sums of rejections are left by launches over rows and sequences: where there are none, no part of a call may
    count on them, and none is asked for. With at most four chunks (V + 7 places in 8192s) there are no such launches."""
    L = pkg._lib.lib()
    size = lambda N, B, V, probs: L.ojx_verify_drafts_workspace(N, B, V, probs)  # noqa: E731
    for V in (10, 32761, 32762, 41000, 1 << 22):
        assert size(0, 3, V, 1) == size(0, 3, V, 0) == 0
        assert size(6, 0, V, 1) == size(6, 0, V, 0) > 0
        assert (size(6, 3, V, 1) > size(6, 3, V, 0)) == (V > 32761)
