"""The attention cores and the paged cache without a GPU: the oracle against closed forms, the mask builder, and what the
entry points refuse before any launch."""
import ctypes
import math

import pytest
import torch

from oracle import cores_oracle as C


# --------------------------------------------------------------------------------------------------------------- oracle
def test_e4m3_table_is_torchs():
    codes = torch.arange(256, dtype=torch.uint8)
    a, b = C.e4m3_table(), codes.view(torch.float8_e4m3fn).double()
    assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))


def test_cache_store_rounds_as_torch_does():
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(64, 128, generator=g) * torch.exp(4 * torch.randn(64, 1, generator=g))).bfloat16()
    x[0], x[1, 3], x[2] = 0, 448.0, (x[2].float() * 1e-38).bfloat16()
    val, scale = C.cache_store(x)
    assert torch.equal(val, (x.double() / scale[:, None]).float().to(torch.float8_e4m3fn).double())
    top = x.double().abs().amax(1) / scale
    assert bool((top <= 448).all()) and bool((top[3:] > 224).all()) and scale[0] == 1 and scale[2] >= 2.0 ** -126


def test_tree_oracle_closed_forms():
    """One position: its value. Equal scores: the mean of the values seen. lse of m equal scores: s + log m."""
    D, page = 128, 16
    kc = torch.zeros(2, 1, page, D, dtype=torch.bfloat16)
    vc = torch.randn(2, 1, page, D, generator=torch.Generator().manual_seed(2)).bfloat16()
    table = torch.tensor([[1, 0]], dtype=torch.int32)
    q = torch.ones(1, 3, D, dtype=torch.bfloat16)
    bits = torch.tensor([[1], [3], [5]])
    o, l, _, _ = C.tree_attn(q, kc, vc, None, None, table, torch.tensor([16]), torch.tensor([0, 3]), bits, 1.0)
    v = torch.cat([vc[1, 0], vc[0, 0]]).double()
    for i, seen in enumerate(([16], [16, 17], [16, 18])):
        rows = list(range(16)) + seen
        assert torch.allclose(o[i, 0], v[rows].mean(0), atol=1e-12) and abs(l[i, 0] - math.log(len(rows))) < 1e-12


def test_linattn_oracle_closed_forms():
    """Without the delta rule: o_t = scale sum e^(G_t - G_j) (q_t . k_j) v_j. With it, beta = 1 and a key of norm 1: the
    state returns the value just written."""
    g = torch.Generator().manual_seed(3)
    R = 9
    q, k, v = (torch.randn(R, 128, generator=g, dtype=torch.float64) for _ in range(3))
    k = k / k.norm(dim=1, keepdim=True)
    gate = -torch.rand(R, 1, generator=g)
    o, st, _, _ = C.linattn(q, k, v, gate, None, [R], None, 0.5)
    G = gate.double().cumsum(0)[:, 0]
    W = torch.exp(G[:, None] - G[None]).tril() * (q @ k.T)
    assert torch.allclose(o[:, 0], 0.5 * W @ v, atol=1e-10)
    o, st, _, _ = C.linattn(q, k, v, gate, torch.ones(R, 1), [R], None, 1.0)
    assert torch.allclose(st[0, 0].T @ k[-1], v[-1], atol=1e-10)


# ------------------------------------------------------------------------------------------------------------ precision
def _pieces(x, n):
    """x, rounded to fp32, as the sum of n bf16 pieces of 8 bits each."""
    left, out = x.float(), torch.zeros_like(x, dtype=torch.float64)
    for _ in range(n):
        piece = left.bfloat16().float()
        left, out = left - piece, out + piece.double()
    return out


def _chunk_in_pieces(q, k, v, g, beta, lengths, state, scale, drop=None, to=1):
    """The chunk's formulas in 64 bits with the factors named in linattn_chunk in their pieces, `drop` in `to`: what a kernel
    with exact sums gives. One key head a value head."""
    R, HV = g.shape
    q, k, v = (x.double().reshape(R, HV, 128) for x in (q, k, v))
    o, st = torch.zeros(R, HV, 128, dtype=torch.float64), torch.zeros(len(lengths), HV, 128, 128, dtype=torch.float64)
    two = lambda x, name: _pieces(x, to if drop == name else 2)  # noqa: E731
    three = lambda x, name: _pieces(x, to if drop == name else 3)  # noqa: E731
    at = 0
    for s, n in enumerate(lengths):
        for h in range(HV):
            r = slice(at, at + n)
            Q, K, V, S0, cum = q[r, h], k[r, h], v[r, h], state[s, h].double(), g[r, h].double().cumsum(0)
            fade = torch.where(torch.ones(n, n).tril() > 0, cum[:, None] - cum[None], -math.inf).exp()
            since, fade_to = cum.exp()[:, None], (cum[-1] - cum).exp()[:, None]
            W = P = fade * (Q @ K.T)
            X, T = V, torch.eye(n, dtype=torch.float64)
            if beta is not None:
                b = beta[r, h].double()
                T = torch.linalg.inv(T + b[:, None] * (fade * (K @ K.T)).tril(-1)) * b[None]
                X, W = V - since * (K @ three(S0, "state of X")), P @ T
                end = three(three(fade_to * T, "T") @ three(X, "X"), "U")
                X = two(X, "X of O")
            else:
                end = three(fade_to * V, "U")
            st[s, h] = since[-1] * S0 + K.T @ end
            o[r, h] = (scale * (since * (Q @ two(S0, "state of O")) + two(W, "P T") @ X)).bfloat16().double()
        at += n
    return o, st


def _short(delta, seed=0):
    """Sequences of 1 to 64 tokens, two heads, states of their own, decays around 1 and slow ones."""
    g = torch.Generator().manual_seed(seed)
    lengths = [1, 2, 3, 5, 8, 16, 24, 40, 64]
    R = sum(lengths)
    qk = torch.nn.functional.silu(torch.randn(2, R, 2, 128, generator=g) + 0.3)
    qk = (qk / qk.norm(dim=-1, keepdim=True)).bfloat16().reshape(2, R, 256)
    v = torch.randn(R, 256, generator=g).bfloat16()
    gate = -torch.rand(R, 2, generator=g) * torch.tensor([1.0, 0.02])
    beta = torch.sigmoid(torch.randn(R, 2, generator=g)).bfloat16() if delta else None
    return (qk[0], qk[1], v, gate, beta), lengths, torch.randn(len(lengths), 2, 128, 128, generator=g)


def test_linattn_chunk_is_linattn():
    for delta in (True, False):
        args, lengths, state = _short(delta)
        a, b = C.linattn(*args, lengths, state, 0.1), C.linattn_chunk(*args, lengths, state, 0.1)
        assert torch.allclose(a[0], b[0], atol=1e-11) and torch.allclose(a[1], b[1], atol=1e-11)


@pytest.mark.parametrize("delta,drop", [(True, x) for x in (None, "state of X", "X", "T", "U", "state of O", "P T", "X of O")]
                         + [(False, x) for x in (None, "U", "state of O", "P T")])
def test_linattn_chunk_bounds_see_a_single_piece(delta, drop):
    """The factors in their pieces stay within the bounds; any one of them in a single piece does not."""
    args, lengths, state = _short(delta, 1)
    o, st, bo, bs = C.linattn_chunk(*args, lengths, state, 128 ** -0.5)
    go, gs = _chunk_in_pieces(*args, lengths, state, 128 ** -0.5, drop)
    worst = max(((go - o).abs() / bo).max().item(), ((gs - st).abs() / bs).max().item())
    assert worst <= 1 if drop is None else worst > 2, worst


def slow_chunks(S, HV, delta, seed):
    """S sequences of 64 tokens that forget little, from states of the size that they keep: q, k, v, g, beta, lengths,
    states. One key head a value head."""
    g = torch.Generator().manual_seed(seed)
    R = S * 64
    qk = torch.nn.functional.silu(torch.randn(2, R, HV, 128, generator=g) + 0.3)
    qk = (qk / qk.norm(dim=-1, keepdim=True)).bfloat16().reshape(2, R, HV * 128)
    v = torch.randn(R, HV * 128, generator=g).bfloat16()
    gate = -0.02 * torch.rand(R, HV, generator=g)
    beta = torch.sigmoid(torch.randn(R, HV, generator=g)).bfloat16() if delta else None
    return (qk[0], qk[1], v, gate, beta), [64] * S, torch.randn(S, HV, 128, 128, generator=g)


# How far an fp32 state may be off, relative to its norm and in half steps of fp32: e^G is off by up to 3 as a whole, and each
# entry stands at the end of a dozen or so of fp32 roundings, 0.6 each in the mean and independent: 2.
STATE_STEPS = 6


@pytest.mark.parametrize("delta,drop", [(True, x) for x in (None, "state of X", "X", "T", "U")] + [(False, None), (False, "U")])
def test_state_steps_see_a_missing_piece(delta, drop):
    """Three pieces of every factor that makes a state are within STATE_STEPS; any one of them in two is past it."""
    args, lengths, state = slow_chunks(2, 2, delta, 1)
    st = C.linattn(*args, lengths, state, 1.0)[1]
    got = _chunk_in_pieces(*args, lengths, state, 1.0, drop, 2)[1]
    steps = (got - st).norm(dim=(2, 3)) / st.norm(dim=(2, 3)) / C.F
    assert bool((steps <= 1).all()) if drop is None else bool((steps > 1.5 * STATE_STEPS).all()), steps


# ----------------------------------------------------------------------------------------------------------------- bits
def test_tree_bits(ext):
    b = ext.tree_bits([[-1, 0, 0, 2, -1], [], [-1]])
    assert b.dtype is torch.int64 and b[:, 0].tolist() == [1, 3, 5, 13, 16, 1]
    long = ext.tree_bits([[j - 1 for j in range(130)]])
    assert tuple(long.shape) == (130, 3)
    for i in (0, 62, 63, 64, 127, 129):
        seen = [j for j in range(192) if (int(long[i, j // 64]) >> (j % 64)) & 1]
        assert seen == list(range(i + 1))
    assert tuple(ext.tree_bits([]).shape) == (0, 1)
    for bad in ([0], [-1, 1], [-2], [-1, 0, 5]):
        with pytest.raises(RuntimeError, match="parents"):
            ext.tree_bits([bad])


# ------------------------------------------------------------------------------------------------------------- refusals
@pytest.fixture()
def p():
    buf = ctypes.create_string_buffer(1 << 12)
    q = ctypes.c_void_p(ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 16)
    q.keep = buf
    return q


def test_cache_refusals(pkg, p):
    L = pkg._lib.lib()
    mis = ctypes.c_void_p(p.value + 2)

    def both(N=3, HKV=2, D=256, fmt=1, pages=4, page=64, k=p, kc=p, ks=p, slots=p):
        return (L.ojx_kv_cache_write(k, p, slots, N, HKV, D, fmt, kc, p, ks, p, pages, page, None),
                L.ojx_kv_cache_read(kc, p, ks, p, slots, N, HKV, D, fmt, k, p, pages, page, None))

    for bad in (dict(D=192), dict(D=0), dict(HKV=0), dict(HKV=2000), dict(page=8), dict(page=40), dict(page=0),
                dict(page=2048), dict(pages=-1), dict(pages=1 << 31), dict(N=-1), dict(N=1 << 31)):
        assert both(**bad) == (2, 2), bad
    for bad in (dict(fmt=2), dict(kc=None), dict(ks=None), dict(k=None), dict(slots=None), dict(k=mis), dict(kc=mis),
                dict(ks=mis), dict(slots=ctypes.c_void_p(p.value + 4))):
        assert both(**bad) == (1, 1), bad
    assert b"aligned" in L.ojx_last_error()
    assert both(N=0, k=None, slots=None) == (0, 0)


def test_tree_refusals(pkg, p):
    L = pkg._lib.lib()
    mis = ctypes.c_void_p(p.value + 4)

    def call(N=4, B=2, HQ=6, HKV=2, D=256, fmt=0, MP=4, pages=8, page=64, q=p, kc=p, ptr=p, ctx=p, table=p, out=p, bits=p,
             words=1, ws=None, nws=0):
        return L.ojx_tree_attn(q, ptr, ctx, bits, words, kc, p, None, None, fmt, table, MP, N, B, HQ, HKV, D, pages, page,
                               0.1, out, None, ws, nws, None)

    for bad in (dict(D=64), dict(HQ=5), dict(HQ=0), dict(HKV=0), dict(HQ=130, HKV=2), dict(N=-1), dict(N=1 << 31),
                dict(B=-1), dict(B=1 << 20), dict(page=24), dict(MP=-1), dict(MP=1 << 26), dict(words=0),
                dict(words=-3), dict(N=1 << 22), dict(pages=-2)):
        assert call(**bad) == 2, bad
    for bad in (dict(fmt=3), dict(fmt=1), dict(q=None), dict(out=None), dict(ptr=None), dict(ctx=None), dict(table=None),
                dict(kc=None), dict(q=mis), dict(out=mis), dict(bits=mis)):
        assert call(**bad) == 1, bad
    assert call(N=0, q=None, out=None) == 0
    assert L.ojx_tree_attn_workspace(4, 2, 5, 2, 256, 4, 64) == -1
    need = L.ojx_tree_attn_workspace(4, 2, 6, 2, 256, 1024, 64)
    assert need >= 0
    if need > 0:
        assert call(MP=1024, ws=p, nws=need - 1) == 3 and call(MP=1024, ws=None, nws=need) == 3


def test_linattn_refusals(pkg, p):
    L = pkg._lib.lib()
    mis = ctypes.c_void_p(p.value + 4)

    def prompt(R=5, S=2, HV=6, HK=2, q=p, k=p, v=p, g=p, ptr=p, state=p, src=p, slots=4, o=p, out=p, ws=None, nws=0):
        return L.ojx_linattn_prompt(q, k, v, g, p, ptr, state, src, slots, R, S, HV, HK, 0.1, o, out, ws, nws, None)

    def step(R=5, HV=6, HK=2, q=p, state=p, slot=p, slots=8, o=p):
        return L.ojx_linattn_step(q, p, p, p, p, state, slot, slots, R, HV, HK, 0.1, o, None)

    for bad in (dict(HV=5), dict(HV=0), dict(HK=0), dict(HV=2048, HK=2), dict(R=-1), dict(R=1 << 31)):
        assert prompt(**bad) == 2 and step(**bad) == 2, bad
    for bad in (dict(S=-1), dict(S=1 << 23), dict(slots=-1), dict(slots=1, src=None)):
        assert prompt(**bad) == 2, bad
    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(g=None), dict(ptr=None), dict(o=None), dict(out=None),
                dict(q=mis), dict(state=mis), dict(out=mis)):
        assert prompt(**bad) == 1, bad
    for bad in (dict(q=None), dict(state=None), dict(slot=None), dict(o=None), dict(state=mis), dict(q=mis)):
        assert step(**bad) == 1, bad
    assert step(R=1 << 22) == 2
    assert step(R=0, q=None, slot=None) == 0
    assert prompt(R=0, S=0, q=None, ptr=None) == 0
    assert L.ojx_linattn_prompt_workspace(5, 2, 5, 2, 1) == -1
    need = L.ojx_linattn_prompt_workspace(5, 2, 6, 2, 1)
    assert need >= 0
    if need > 0:
        assert prompt(ws=p, nws=need - 1) == 3 and prompt(ws=None, nws=need) == 3


def test_refusals_of_sizes_whose_products_wrap(pkg, p):
    """Page and sequence counts whose products with the other sizes come back to something small in 64 bits."""
    L = pkg._lib.lib()
    for MP, page in ((1 << 60, 16), (1 << 58, 64), ((1 << 60) + 1, 16), (1 << 62, 1024)):
        assert L.ojx_tree_attn_workspace(4, 2, 6, 2, 256, MP, page) == -1
        assert L.ojx_tree_attn(p, p, p, None, 0, p, p, None, None, 0, p, MP, 4, 2, 6, 2, 256, 8, page, 0.1, p, None, None, 0,
                               None) == 2
    for S in (1 << 61, (1 << 61) - 1, (1 << 62) - 1, (1 << 63) - 1, 1 << 31):
        for HV, HK in ((6, 2), (1, 1), (1024, 16)):
            assert L.ojx_linattn_prompt_workspace(5, S, HV, HK, 1) == -1
            assert L.ojx_linattn_prompt(p, p, p, p, p, p, None, None, 0, 5, S, HV, HK, 0.1, p, p, p, 1 << 40, None) == 2


def test_python_refusals(ext):
    """CPU tensors are refused like everywhere in the package."""
    x = torch.zeros(2, 3, 256, dtype=torch.bfloat16)
    kc = torch.zeros(4, 2, 16, 256, dtype=torch.bfloat16)
    i32, i64 = torch.zeros(3, dtype=torch.int32), torch.zeros(3, dtype=torch.int64)
    for call in (lambda: ext.kv_cache_write(x, x, i64, kc, kc), lambda: ext.kv_cache_read(kc, kc, i64),
                 lambda: ext.tree_attn(x, kc, kc, i32[None], i32[:1], i32[:2]),
                 lambda: ext.linattn_prompt(x[0], x[0], x[0], x[0, :, :2].float(), None, i32),
                 lambda: ext.linattn_step(x[0], x[0], x[0], x[0, :, :2].float(), None, kc.float(), i32)):
        with pytest.raises(RuntimeError, match="contiguous CUDA"):
            call()


def test_python_refusals_of_shapes(ext, monkeypatch):
    """Everything a kernel would read past is refused by its shape, before the library is called. (Tensors on the CPU pass
    the device checks here; the library must not be reached.)"""
    class Lib:
        def __getattr__(self, name):
            raise AssertionError(f"{name} was called")

    monkeypatch.setattr(ext, "_chk", lambda t, name, dtype=None: None if t is not None and t.is_contiguous() and (
        dtype is None or t.dtype is dtype) else (_ for _ in ()).throw(RuntimeError(f"{name}")))
    monkeypatch.setattr(ext, "_one_device", lambda *a: None)
    monkeypatch.setattr(ext, "lib", Lib)
    z = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t)  # noqa: E731
    f, i32, i64, e8 = torch.float32, torch.int32, torch.int64, torch.float8_e4m3fn
    kc, k8, sc = z(4, 2, 16, 256), z(4, 2, 16, 256, t=torch.uint8).view(e8), z(4, 2, 16, t=f)
    x, at = z(2, 3, 256), z(3, t=i64)
    for bad in (lambda: ext.kv_cache_write(x, z(2, 4, 256), at, kc, kc), lambda: ext.kv_cache_write(x, x, at[:2], kc, kc),
                lambda: ext.kv_cache_write(z(3, 3, 256), z(3, 3, 256), at, kc, kc),
                lambda: ext.kv_cache_write(x, x, at, kc, z(4, 2, 32, 256)), lambda: ext.kv_cache_write(x, x, at, k8, k8),
                lambda: ext.kv_cache_write(x, x, at, k8, k8, sc, sc[:3]), lambda: ext.kv_cache_write(x, x, at, kc, kc, sc, sc),
                lambda: ext.kv_cache_write(x, x, at, kc, k8, sc, sc), lambda: ext.kv_cache_write(x, x, at.int(), kc, kc),
                lambda: ext.kv_cache_write(x, x, at, kc.float(), kc.float()),
                lambda: ext.kv_cache_write(z(2, 2, 3, 256), z(2, 2, 3, 256), at, kc, kc),
                lambda: ext.kv_cache_read(kc[0], kc[0], at), lambda: ext.kv_cache_read(k8, k8, at, sc),
                lambda: ext.kv_cache_read(kc, kc, at.int())):
        with pytest.raises(RuntimeError):
            bad()
    q, table, ctx, ptr, bits = z(6, 3, 256), z(1, 4, t=i32), z(1, t=i32), z(2, t=i32), z(3, 1, t=i64)
    for bad in (lambda: ext.tree_attn(z(5, 3, 256), kc, kc, table, ctx, ptr), lambda: ext.tree_attn(z(6, 3, 128), kc, kc, table, ctx, ptr),
                lambda: ext.tree_attn(q, kc, kc, table[0], ctx, ptr), lambda: ext.tree_attn(q, kc, kc, z(2, 4, t=i32), ctx, ptr),
                lambda: ext.tree_attn(q, kc, kc, table, ctx, z(3, t=i32)), lambda: ext.tree_attn(q, kc, kc, table, ctx, ptr, bits[:2]),
                lambda: ext.tree_attn(q, kc, kc, table, ctx, ptr, bits[:, :0]), lambda: ext.tree_attn(q, kc, kc, table, ctx, ptr, bits[:, 0]),
                lambda: ext.tree_attn(q, kc, kc, table.long(), ctx, ptr), lambda: ext.tree_attn(q, k8, k8, table, ctx, ptr)):
        with pytest.raises(RuntimeError):
            bad()
    y, v, g, b, sp = z(5, 256), z(5, 768), z(5, 6, t=f), z(5, 6), z(3, t=i32)
    st, src = z(4, 6, 128, 128, t=f), z(2, t=i32)
    ok = (y, y, v, g, b)
    for bad in (lambda: ext.linattn_prompt(z(5, 200), z(5, 200), v, g, b, sp), lambda: ext.linattn_prompt(y, z(5, 128), v, g, b, sp),
                lambda: ext.linattn_prompt(y, y, z(5, 512), g, b, sp), lambda: ext.linattn_prompt(y, y, v, g[:4], b, sp),
                lambda: ext.linattn_prompt(y, y, v, g, b[:4], sp), lambda: ext.linattn_prompt(y, y, z(5, 640), z(5, 5, t=f), None, sp),
                lambda: ext.linattn_prompt(*ok, sp[:0]), lambda: ext.linattn_prompt(*ok, sp, st),
                lambda: ext.linattn_prompt(*ok, sp, st[:, :5], src), lambda: ext.linattn_prompt(*ok, sp, st, src[:1]),
                lambda: ext.linattn_prompt(*ok, sp, None, src), lambda: ext.linattn_prompt(*ok, sp.long()),
                lambda: ext.linattn_step(*ok, st, z(4, t=i32)), lambda: ext.linattn_step(*ok, st[0], z(5, t=i32)),
                lambda: ext.linattn_step(*ok, st, z(5, t=i64)), lambda: ext.linattn_step(y, y, v, g.bfloat16(), b, st, z(5, t=i32))):
        with pytest.raises(RuntimeError):
            bad()
