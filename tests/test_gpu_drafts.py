"""GPU parity of the operators around drafted tokens (ext.verify_drafts, linattn_tree, linattn_keep, kv_cache_keep,
kv_pages_resize, kv_pages_fork, kv_pages_copy) with the 64-bit oracle (oracle/drafts_oracle.py): whole numbers and copies
equal, linear attention within the oracle's bounds."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32


def _say(*a):
    print(*a, flush=True)


@pytest.fixture(scope="module")
def D():
    from oracle import drafts_oracle
    return drafts_oracle


def _put(dev, *ts):
    return [None if t is None else t.to(dev) for t in ts]


def _ptr(lengths, lead=0):
    return torch.tensor([lead] + [lead + sum(lengths[:i + 1]) for i in range(len(lengths))], dtype=I32)


def _parents(lengths, kind, g):
    """Rows followed: "line", "star" (all behind row 0), "wide" (any earlier row), "near" (one of the last three)."""
    out = []
    for n in lengths:
        for j in range(n):
            low = {"line": j - 1, "star": 0, "wide": 0, "near": max(0, j - 3)}[kind]
            high = {"line": j - 1, "star": 0, "wide": j - 1, "near": j - 1}[kind]
            out.append(-1 if j == 0 else int(torch.randint(low, high + 1, (1,), generator=g)))
    return torch.tensor(out, dtype=I32)


# --------------------------------------------------------------------------------------------------------------- verify
def _verify_case(lengths, V, dtype=BF16, probs="none", kind="near", pad=0, seed=0, spare=0, lead=0, temps=None, near=0.6):
    """Peaked logits, a draft near the target and tokens drawn from it, so that paths of all lengths come up."""
    g = torch.Generator().manual_seed(seed)
    N = lead + sum(lengths) + spare
    raw = 1.5 * torch.randn(N, V + pad, generator=g)
    for _ in range(min(6, V)):
        raw.scatter_(1, torch.randint(0, V, (N, 1), generator=g), 4.0 + 5.0 * torch.rand(N, 1, generator=g))
    logits = raw.to(dtype)[:, pad // 2:pad // 2 + V]
    B = len(lengths)
    temp = torch.tensor(temps if temps is not None else [(1.0, 0.7, 0.0, 1.3)[b % 4] for b in range(B)])
    tree = torch.cat([torch.full((lead,), -1, dtype=I32), _parents(lengths, kind, g), torch.full((spare,), -1, dtype=I32)])
    q = torch.softmax(raw[:, pad // 2:pad // 2 + V] + near * torch.randn(N, V, generator=g), -1)
    tokens = torch.zeros(N, dtype=torch.int64)
    at = lead
    for n in lengths:
        for j in range(n):
            tokens[at + j] = int(torch.multinomial(q[at + max(0, int(tree[at + j]))], 1, generator=g))
        at += n
    return {"logits": logits, "tokens": tokens, "q_ptr": _ptr(lengths, lead), "u": torch.rand(N, generator=g),
            "parents": None if kind == "line" else tree,
            "probs": {"none": None, "bf16": q.bfloat16(), "fp32": q}[probs], "temperature": temp}


def _strided(t, dev):
    """t on the GPU with the row stride (and the first row's offset) it has on the CPU."""
    if t is None or t.is_contiguous():
        return None if t is None else t.to(dev)
    back = torch.empty(t.shape[0] * t.stride(0) + t.storage_offset(), dtype=t.dtype, device=dev)
    out = back.as_strided(t.shape, t.stride(), t.storage_offset())
    out.copy_(t)
    return out


def _run_verify(ext, c, dev):
    d = {x: _strided(t, dev) for x, t in c.items()}
    return [t.cpu() for t in ext.verify_drafts(d["logits"], d["tokens"], d["q_ptr"], d["u"], d["parents"], d["probs"],
                                               d["temperature"])]


def _check_verify(D, c, got, least=1e-11):
    path, count, nxt, near = D.verify(**{x: (t.tolist() if x in ("q_ptr", "tokens") else t) for x, t in c.items()})
    assert near > least, f"a test lies {near:.1e} from its border: choose another seed"
    assert got[1].tolist() == count
    assert got[0].tolist() == path
    assert got[2].tolist() == nxt
    return count


VERIFY = [
    # rows, V, type, pad
    ([1], 1, F32, 0), ([2], 2, BF16, 0), ([6], 1000, BF16, 0), ([5, 0, 3, 1, 4], 37, F32, 3),
    ([4, 7, 2], 8185, BF16, 0), ([3, 9], 8192, BF16, 5), ([5, 5], 8193, F32, 0), ([6, 3, 8, 2, 2], 20011, BF16, 1),
    ([12] * 9, 16385, BF16, 0), ([70, 3], 301, F32, 2), ([130, 1, 66], 50, BF16, 0),
]


@pytest.mark.parametrize("kind", ["line", "near", "star", "wide"])
@pytest.mark.parametrize("probs", ["none", "bf16", "fp32"])
@pytest.mark.parametrize("case", range(len(VERIFY)))
def test_verify(ext, D, dev, case, probs, kind):
    lengths, V, dtype, pad = VERIFY[case]
    _say(f"case verify {case} probs={probs} {kind}")
    c = _verify_case(lengths, V, dtype, probs, kind, pad, seed=case * 31 + len(kind))
    count = _check_verify(D, c, _run_verify(ext, c, dev))
    _say(f"  accepted {count}")


@pytest.mark.parametrize("probs", ["none", "fp32"])
def test_verify_many_rejections(ext, D, dev, probs):
    """A draft far from the target, children of one row in dozens: rejections beyond those that the whole chip sums."""
    for seed in range(4):
        c = _verify_case([40, 25, 64, 90], 9000, BF16, probs, "star", seed=seed, near=6.0, temps=[1.0, 0.5, 2.0, 1.0])
        _check_verify(D, c, _run_verify(ext, c, dev))
        c = _verify_case([40, 25, 64, 90], 9000, BF16, probs, "wide", seed=seed, near=4.0, temps=[1.0, 0.5, 2.0, 1.0])
        _check_verify(D, c, _run_verify(ext, c, dev))


@pytest.mark.parametrize("dtype,V,pad", [(BF16, 16500, 3), (F32, 9001, 0)])
def test_verify_many_rows(ext, D, dev, dtype, V, pad):
    """Enough rows that a workgroup takes several chunks of one, the last of them alone; unaligned rows."""
    c = _verify_case([7, 0, 9, 5] * 200, V, dtype, "none", "near", pad, seed=12)
    _check_verify(D, c, _run_verify(ext, c, dev))


@pytest.mark.parametrize("probs", ["none", "bf16", "fp32"])
def test_verify_temperatures(ext, D, dev, probs):
    temps = [0.0, -1.0, math.nan, math.inf, 1e-3, 1e-40, 50.0, 1.0]
    c = _verify_case([6] * 8, 700, BF16, probs, "near", seed=5, temps=temps)
    _check_verify(D, c, _run_verify(ext, c, dev))
    c["temperature"] = None
    _check_verify(D, c, _run_verify(ext, c, dev))


@pytest.mark.parametrize("probs", ["none", "fp32"])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_verify_masks(ext, D, dev, dtype, probs):
    """Logits of -infinity and of the type's lowest value, rows of nothing else, NaN and +infinity, each somewhere on the
    way and at its end; tokens and parents that are none."""
    low = torch.finfo(dtype).min
    for seed in range(6):
        c = _verify_case([7] * 12, 8200, dtype, probs, "near", seed=seed, temps=[1.0, 0.0, 0.8] * 4)
        x, P = c["logits"], c["parents"]
        x[0:28, 100:] = -math.inf
        x[7:14, ::2] = low
        x[14:21, 50:] = low
        x[21 + seed, :] = -math.inf
        x[28 + seed, 8199] = math.nan
        x[35 + seed, 3] = math.inf
        x[42, :] = -math.inf
        x[49, :] = math.nan
        x[56, :] = low
        x[63:70] = -math.inf
        x[63:70, 8198] = low
        c["tokens"][70:77] = torch.tensor([0, -1, 8200, 1 << 40, -(1 << 40), 8199, 0])
        P[77:84] = torch.tensor([5, 1, 7, -3, 0, 100, 3])
        _check_verify(D, c, _run_verify(ext, c, dev))


@pytest.mark.parametrize("probs", ["none", "fp32"])
def test_verify_same_token_again(ext, D, dev, probs):
    """Children of one row with the same token: once rejected, it is gone, unless draws from q may repeat it."""
    c = _verify_case([9] * 16, 12, F32, probs, "star", seed=3, temps=[1.0, 0.0] * 8)
    c["tokens"] = c["tokens"] % 3
    _check_verify(D, c, _run_verify(ext, c, dev))


def test_verify_borders(ext, dev):
    """Numbers on the borders themselves, where every sum is exact."""
    logits = torch.tensor([[0.0, 0.0, 0.0, -math.inf, 0.0]]).repeat(2, 1).bfloat16()       # 1/4 each, but for one
    c = {"logits": logits, "tokens": torch.tensor([0, 2]), "q_ptr": torch.tensor([0, 2], dtype=I32), "parents": None,
         "probs": None, "temperature": None}
    low = 0.25 - 2.0 ** -26
    for u, count, nxt in (((0.0, 0.0), 2, 0), ((0.25, low), 2, 1), ((low, 0.25), 1, 0), ((0.75, 0.0), 2, 4),
                          ((1 / 3, 0.5), 1, 1), ((0.999, 0.999), 1, 4), ((1.0, 1.0), 1, 4), ((math.nan, math.nan), 1, 4),
                          ((-1.0, -1.0), 2, 0), ((0.5, 0.0), 2, 2)):
        got = _run_verify(ext, {**c, "u": torch.tensor(u)}, dev)
        assert got[1].tolist() == [count] and got[2].tolist() == [nxt], u
    # q twice p there, and none elsewhere: accepted up to one half
    q = torch.tensor([[0.0, 0.0, 0.5, 0.0, 0.5]]).repeat(2, 1)
    for u, count, nxt in (((0.3, 0.499), 2, 1), ((0.0, 0.5), 1, 0), ((0.499, 0.5), 1, 0), ((0.5, 0.5), 1, 1)):
        got = _run_verify(ext, {**c, "probs": q, "u": torch.tensor(u)}, dev)
        assert got[1].tolist() == [count] and got[2].tolist() == [nxt], u
    # nothing left of p: drawn from p; a draft that never proposes what it proposed
    same = torch.tensor([[0.25, 0.25, 0.25, 0.0, 0.25]]).repeat(2, 1)
    assert _run_verify(ext, {**c, "probs": same, "u": torch.tensor([0.6, 1.0])}, dev)[2].tolist() == [2]
    for bad in (0.0, -1.0, math.nan):
        q0 = torch.full((2, 5), bad)
        assert _run_verify(ext, {**c, "probs": q0, "u": torch.tensor([0.3, 0.9])}, dev)[1].tolist() == [2]


@pytest.mark.parametrize("V", [9000, 41000])
def test_verify_chunks_with_nothing_left(ext, dev, V):
    """A random number of 0 passes over all that is masked, rejected or proposed more often than wanted."""
    at = [5, 8500, 8600, V - 1]
    logits = torch.full((2, V), -math.inf)
    logits[:, at] = 0.0                                                       # 1/4 each
    c = {"logits": logits, "q_ptr": torch.tensor([0, 2], dtype=I32), "parents": None, "temperature": None}
    got = _run_verify(ext, {**c, "probs": None, "tokens": torch.tensor([0, 5]), "u": torch.tensor([0.0, 0.25])}, dev)
    assert got[1].tolist() == [1] and got[2].tolist() == [8500]
    q = torch.zeros(2, V)
    q[:, at[:2]] = 0.5
    tree = torch.tensor([-1, 0], dtype=I32)
    for parents in (None, tree):
        d = {**c, "probs": q, "tokens": torch.tensor([0, 8500]), "parents": parents}
        assert _run_verify(ext, {**d, "u": torch.tensor([0.0, 0.5])}, dev)[2].tolist() == [8600]
        assert _run_verify(ext, {**d, "u": torch.tensor([0.5, 0.5])}, dev)[2].tolist() == [V - 1]
        d["probs"] = torch.where(q > 0, 1.0, 0.25 * torch.isfinite(logits))      # as often as wanted, or more: nothing left
        got = _run_verify(ext, {**d, "u": torch.tensor([0.0, 0.25])}, dev)
        assert got[1].tolist() == [1] and got[2].tolist() == [5]
        assert _run_verify(ext, {**d, "u": torch.tensor([0.75, 0.25])}, dev)[2].tolist() == [V - 1]


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("kind", ["line", "star", "near"])
def test_verified_tokens_are_the_targets(ext, dev, kind, probs):
    """Over 60000 sequences the first token that comes out is distributed as the target's: each count within five standard
    deviations (a chance of 6e-7 for each of some 100 counts)."""
    B, n, V = 60000, 4, 9
    g = torch.Generator(device=dev).manual_seed(7 + len(kind))
    row = torch.randn(n, V, generator=g, device=dev) * 1.5
    logits = row.repeat(B, 1)
    q = torch.softmax(row + torch.randn(n, V, generator=g, device=dev), -1)
    parents = {"line": [-1, 0, 1, 2], "star": [-1, 0, 0, 0], "near": [-1, 0, 0, 1]}[kind]
    up = torch.tensor([max(0, x) for x in parents], device=dev)
    if probs:
        tokens = torch.multinomial(q[up].repeat(B, 1), 1, generator=g)[:, 0]
    else:
        tokens = torch.tensor([0, 1, 4, 1], device=dev).repeat(B)
    u = torch.rand(B * n, generator=g, device=dev)
    ptr = torch.arange(0, B * n + 1, n, dtype=I32, device=dev)
    tree = None if kind == "line" else torch.tensor(parents, dtype=I32, device=dev).repeat(B)
    path, count, nxt = ext.verify_drafts(logits, tokens, ptr, u, tree, q.repeat(B, 1) if probs else None)
    path, at = path.reshape(B, n), torch.arange(B, device=dev)
    child = path[:, 1].clamp_min(0).long()
    first = torch.where(count > 1, tokens[at * n + child], nxt)
    p = torch.softmax(row[0].double(), 0)
    seen = torch.bincount(first, minlength=V).double()
    assert bool(((seen - B * p).abs() <= 5 * (B * p * (1 - p)).sqrt() + 1).all()), (seen / B, p)
    # and the second, behind each first token of the line that was accepted
    if kind == "line":
        p2 = torch.softmax(row[1].double(), 0)
        some = count > 1
        second = torch.where(count > 2, tokens[at * n + 2], nxt)[some]
        m = int(some.sum())
        seen = torch.bincount(second, minlength=V).double()
        assert bool(((seen - m * p2).abs() <= 5 * (m * p2 * (1 - p2)).sqrt() + 1).all()), (seen / m, p2)


@pytest.mark.parametrize("probs", ["none", "fp32"])
def test_verify_rows_of_no_sequence(ext, D, dev, probs):
    c = _verify_case([3, 4], 100, BF16, probs, "near", seed=2, lead=2, spare=5)
    got = _run_verify(ext, c, dev)
    _check_verify(D, c, got)
    for ptr in ([9, 2, 5], [-4, 3, 2], [0, 100, 3], [2, 2, 2]):                   # falling, outside, empty
        c["q_ptr"] = torch.tensor(ptr, dtype=I32)
        _check_verify(D, c, _run_verify(ext, c, dev))


def test_verify_empty(ext, dev):
    e = lambda *s, t=I32: torch.empty(*s, dtype=t, device=dev)  # noqa: E731
    path, count, nxt = ext.verify_drafts(e(0, 10, t=F32), e(0, t=torch.int64), torch.zeros(4, dtype=I32, device=dev), e(0, t=F32))
    assert path.shape == (0,) and count.tolist() == [0] * 3 and nxt.tolist() == [-1] * 3
    path, count, nxt = ext.verify_drafts(torch.zeros(3, 10, device=dev), torch.zeros(3, dtype=torch.int64, device=dev),
                                         torch.zeros(1, dtype=I32, device=dev), torch.zeros(3, device=dev))
    assert path.tolist() == [-1] * 3 and count.shape == (0,)


def test_verify_largest_vocabulary(ext, D, dev):
    V = 1 << 22
    c = _verify_case([2], V, BF16, "none", "line", seed=4, temps=[1.0])
    c["u"][1] = 0.9999
    _check_verify(D, c, _run_verify(ext, c, dev), least=1e-13)
    with pytest.raises(RuntimeError, match="bad sizes"):
        ext.verify_drafts(torch.zeros(1, V + 1, device=dev), torch.zeros(1, dtype=torch.int64, device=dev),
                          torch.tensor([0, 1], dtype=I32, device=dev), torch.zeros(1, device=dev))


@pytest.mark.parametrize("probs", ["none", "fp32"])
def test_verify_past_32_bits(ext, D, dev, probs):
    """Rows whose byte offsets pass 2^32 and element offsets 2^31."""
    c = _verify_case([5], 3000, BF16, probs, "near", seed=6, temps=[0.9])
    want = _run_verify(ext, c, dev)
    _check_verify(D, c, want)
    ld = (1 << 29) + 17
    d = {x: None if t is None else t.to(dev) for x, t in c.items()}
    for name in ("logits", "probs"):
        if d[name] is not None:
            back = torch.empty(4 * ld + 3000, dtype=d[name].dtype, device=dev)
            far = back.as_strided((5, 3000), (ld, 1))
            far.copy_(d[name])
            d[name] = far
    got = ext.verify_drafts(d["logits"], d["tokens"], d["q_ptr"], d["u"], d["parents"], d["probs"], d["temperature"])
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)


def test_verify_logits_of_a_projection(ext, D, dev):
    """Logits as they leave the package's own projection, wider than the vocabulary."""
    g = torch.Generator().manual_seed(8)
    x, w = torch.randn(9, 64, generator=g).bfloat16().to(dev), (0.6 * torch.randn(1008, 64, generator=g)).bfloat16().to(dev)
    logits = ext.mm(x, w)[:, :1001]
    c = _verify_case([4, 5], 1001, BF16, "fp32", "near", seed=9, temps=[1.0, 0.6])
    c["logits"] = logits.cpu()
    c["tokens"][1], c["tokens"][5] = int(c["logits"][0].argmax()), int(c["logits"][4].argmax())
    d = {k: None if t is None else t.to(dev) for k, t in c.items()}
    got = ext.verify_drafts(logits, d["tokens"], d["q_ptr"], d["u"], d["parents"], d["probs"], d["temperature"])
    _check_verify(D, c, [t.cpu() for t in got])


# ----------------------------------------------------------------------------------------------------- linear attention
def _lin_case(N, HK, G, delta, seed, sharp=False):
    g = torch.Generator().manual_seed(seed)
    HV = HK * G
    qk = torch.nn.functional.silu(torch.randn(2, N, HK, 128, generator=g) + 0.3)
    if sharp and N > 3:
        qk[1, 1::3] = qk[1, :1]
    qk = (qk / (qk.square().sum(-1, keepdim=True) + 1e-6).sqrt()).bfloat16().reshape(2, N, HK * 128)
    v = torch.nn.functional.silu(torch.randn(N, HV * 128, generator=g)).bfloat16()
    gate = -torch.rand(N, HV, generator=g) * torch.exp(3 * torch.randn(HV, generator=g) - 2)
    beta = torch.sigmoid(2 * torch.randn(N, HV, generator=g)).bfloat16()
    if sharp:
        pick = torch.rand(N, HV, generator=g)
        gate = torch.where(pick < 0.3, torch.zeros(()), gate)
        gate = torch.where(pick > 0.97, torch.full((), -math.inf), torch.where(pick > 0.94, torch.full((), -150.0), gate))
        beta = torch.where(torch.rand(N, HV, generator=g) < 0.2, torch.ones(()), beta.float()).bfloat16()
        beta = torch.where(torch.rand(N, HV, generator=g) < 0.2, torch.zeros(()), beta.float()).bfloat16()
    return qk[0].contiguous(), qk[1].contiguous(), v, gate, beta if delta else None


def _check_tree(D, args, state, slot, ptr, parents, scale, got):
    o, bo = D.linattn_tree(*args, state, slot.tolist(), ptr.tolist(), parents, scale)
    got = got.cpu().double().reshape(o.shape)
    none = torch.isnan(o)
    assert torch.equal(none, torch.isnan(got))
    err = torch.where(none, 0.0, (got - o).abs())
    worst = (err / bo.clamp_min(1e-300)).max().item() if o.numel() else 0.0
    _say(f"  out {worst:.3f} of its bound")
    assert bool((err <= bo).all()), f"out: {worst:.3f} of the bound"


TREES = [
    # rows, HK, G
    ([1], 1, 1), ([2], 2, 3), ([5, 0, 3], 1, 2), ([16], 2, 1), ([17, 15], 1, 3), ([12] * 5, 2, 3), ([33, 48, 7], 1, 1),
    ([64], 1, 3), ([63, 1, 40], 2, 1),
]


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("kind", ["line", "near", "star", "wide"])
@pytest.mark.parametrize("case", range(len(TREES)))
def test_tree(ext, D, dev, case, kind, delta):
    lengths, HK, G = TREES[case]
    _say(f"case tree {case} {kind} delta={delta}")
    g = torch.Generator().manual_seed(case)
    N, B = sum(lengths), len(lengths)
    args = _lin_case(N, HK, G, delta, seed=case, sharp=case % 2 == 1)
    parents = None if kind == "line" else _parents(lengths, kind, g)
    state = 0.3 * torch.randn(B + 2, HK * G, 128, 128, generator=g)
    slot = torch.randperm(B + 2, generator=g)[:B].int()
    ptr = _ptr(lengths)
    d = _put(dev, *args, state, slot, ptr, parents)
    keep = d[5].clone()
    got = ext.linattn_tree(*d, scale=0.2)
    assert torch.equal(d[5], keep)
    _check_tree(D, args, state, slot, ptr, parents, 0.2, got)


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("lengths,kind", [([65], "line"), ([130, 3], "near"), ([200], "wide"), ([64, 300], "star")])
def test_tree_of_many_rows(ext, D, dev, lengths, kind, delta):
    _say(f"case long tree {lengths} {kind} delta={delta}")
    g = torch.Generator().manual_seed(len(lengths))
    N, B = sum(lengths), len(lengths)
    args = _lin_case(N, 1, 1, delta, seed=N)
    parents = None if kind == "line" else _parents(lengths, kind, g)
    state, slot, ptr = 0.3 * torch.randn(B, 1, 128, 128, generator=g), torch.arange(B, dtype=I32), _ptr(lengths)
    got = ext.linattn_tree(*_put(dev, *args, state, slot, ptr, parents))
    _check_tree(D, args, state, slot, ptr, parents, 128 ** -0.5, got)


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("n", [7, 30])
def test_tree_odd_parents_slots_and_pointers(ext, D, dev, n, delta):
    """Several rows on the state itself, parents that are none, slots shared, idle and outside, rows of no sequence."""
    g = torch.Generator().manual_seed(n)
    lengths = [n, n, 3, 4, n]
    N = 2 + sum(lengths) + 3
    args = _lin_case(N, 1, 2, delta, seed=n)
    parents = torch.cat([torch.full((2,), 7, dtype=I32), _parents(lengths, "wide", g), torch.zeros(3, dtype=I32)])
    parents[4], parents[5], parents[6] = -1, -9, 100
    parents[2 + n:2 + 2 * n] = torch.arange(n, dtype=I32)                            # every row its own: on the state
    state, slot = 0.3 * torch.randn(3, 2, 128, 128, generator=g), torch.tensor([1, 1, -2, 3, 1 << 30], dtype=I32)
    for ptr in (_ptr(lengths, 2), torch.tensor([4, 9, 6, 12, -1, 2000], dtype=I32)):
        got = ext.linattn_tree(*_put(dev, *args, state, slot, ptr, parents))
        _check_tree(D, args, state, slot, ptr, parents, 128 ** -0.5, got)
    slot[:] = 0
    got = ext.linattn_tree(*_put(dev, *args, state, slot, ptr, parents))
    _check_tree(D, args, state, slot, ptr, parents, 128 ** -0.5, got)


@pytest.mark.parametrize("delta", [True, False])
def test_tree_long_sequences_among_others(ext, D, dev, delta):
    """Sequences of more than 64 rows beside short, empty, idle ones and one whose state is not there; falling pointers."""
    g = torch.Generator().manual_seed(6)
    lengths = [70, 3, 0, 130, 64, 90, 65]
    N = sum(lengths) + 5
    args = _lin_case(N, 1, 2, delta, seed=6)
    parents = torch.cat([_parents(lengths, "near", g), torch.zeros(5, dtype=I32)])
    parents[69], parents[80] = -1, 500
    state = 0.3 * torch.randn(3, 2, 128, 128, generator=g)
    slot = torch.tensor([1, -1, 0, 0, 2, 7, 2], dtype=I32)
    for ptr in (_ptr(lengths), torch.tensor([2, 70, 60, 260, 200, 380, 390, 5], dtype=I32)):
        d = _put(dev, *args, state, slot, ptr, parents)
        got = ext.linattn_tree(*d)
        assert torch.equal(got, ext.linattn_tree(*d)) or bool(torch.isnan(got).any())
        _check_tree(D, args, state, slot, ptr, parents, 128 ** -0.5, got)


def _below(parents, n, j):
    """Rows of a sequence that hang on row j, itself among them."""
    out = {j}
    for i in range(j + 1, n):
        if int(parents[i]) in out and int(parents[i]) < i:
            out.add(i)
    return sorted(out)


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("n", [9, 40, 90])
@pytest.mark.parametrize("what", ["k", "v", "beta", "g", "+g", "q"])
def test_tree_values_not_finite(ext, D, dev, what, n, delta):
    """NaN or an infinity in one row reaches the rows that hang on it (a query: the row alone) and no other bit."""
    if what == "beta" and not delta:
        return
    _say(f"case not finite {what} n={n} delta={delta}")
    g = torch.Generator().manual_seed(n)
    HV = 3
    q, k, v, gate, beta = _lin_case(n, 1, 3, delta, seed=n)
    parents = _parents([n], "near", g)
    state, slot, ptr = 0.3 * torch.randn(1, HV, 128, 128, generator=g), torch.zeros(1, dtype=I32), _ptr([n])
    clean = ext.linattn_tree(*_put(dev, q, k, v, gate, beta, state, slot, ptr, parents)).cpu().reshape(n, HV, 128)
    free, bo = D.linattn_tree(q, k, v, gate, beta, state, [0], [0, n], parents, 128 ** -0.5)
    j = n // 3
    if what == "k":
        k[j, 5] = math.nan
    elif what == "q":
        q[j, 5] = math.inf
    elif what == "v":
        v[j, 128 + 7] = math.inf
    elif what == "beta":
        beta[j, 1] = math.nan
    else:
        gate[j, 1] = math.nan if what == "g" else math.inf
    got = ext.linattn_tree(*_put(dev, q, k, v, gate, beta, state, slot, ptr, parents)).cpu().reshape(n, HV, 128)
    hit = [j] if what == "q" else _below(parents, n, j)
    rest = [i for i in range(n) if i not in hit]
    o = D.linattn_tree(q, k, v, gate, beta, state, [0], [0, n], parents, 128 ** -0.5)[0]
    for h in range(HV):
        one = what in ("k", "q") or h == 1
        assert bool(((got[rest, h].double() - free[rest, h]).abs() <= bo[rest, h]).all())
        if one:
            bad = slice(7, 8) if what == "v" else slice(None)
            for i in hit:
                # a child may not see it (a strength of zero for the row, a decay to nothing): as the definition has it
                want = torch.isfinite(o[i, h, bad])
                assert torch.equal(torch.isfinite(got[i, h, bad]), want), (h, i)
                if what == "v":
                    others = [x for x in range(128) if x != 7]
                    assert bool((got[i, h, others].double() - clean[i, h, others].double()).abs().max() <= 0.02)
        else:
            assert torch.equal(got[:, h], clean[:, h])


def test_tree_state_not_finite(ext, D, dev):
    """NaN or an infinity in a state stays in its value dim of its head."""
    n = 20
    g = torch.Generator().manual_seed(3)
    args = _lin_case(n, 1, 3, True, seed=3)
    parents, slot, ptr = _parents([n], "near", g), torch.zeros(1, dtype=I32), _ptr([n])
    state = 0.3 * torch.randn(1, 3, 128, 128, generator=g)
    clean = ext.linattn_tree(*_put(dev, *args, state, slot, ptr, parents)).cpu().reshape(n, 3, 128)
    state[0, 1, 4, 9], state[0, 1, 90, 77] = math.nan, math.inf
    got = ext.linattn_tree(*_put(dev, *args, state, slot, ptr, parents)).cpu().reshape(n, 3, 128)
    assert torch.equal(got[:, [0, 2]], clean[:, [0, 2]])
    others = [x for x in range(128) if x not in (9, 77)]
    assert not bool(torch.isfinite(got[:, 1, 9].float()).any()) and not bool(torch.isfinite(got[:, 1, 77].float()).any())
    assert bool((got[:, 1, others].float() - clean[:, 1, others].float()).abs().max() <= 0.02)


@pytest.mark.parametrize("n", [1, 20, 90])
def test_tree_state_past_16_bits(ext, D, dev, n):
    """Without the delta rule too, infinities in a state come out as such, and what rounds to one in 16 bits as it is."""
    g = torch.Generator().manual_seed(n)
    args = _lin_case(n, 1, 2, False, seed=n)
    parents, slot, ptr = _parents([n], "near", g), torch.zeros(1, dtype=I32), _ptr([n])
    state = 0.3 * torch.randn(1, 2, 128, 128, generator=g)
    state[0, 1, 90, 77], state[0, 1, 3, 20] = math.inf, torch.finfo(F32).max
    got = ext.linattn_tree(*_put(dev, *args, state, slot, ptr, parents)).cpu().double().reshape(n, 2, 128)
    o, bo = D.linattn_tree(*args, state, [0], [0, n], parents, 128 ** -0.5)
    assert bool(torch.isinf(o[:, 1, 77]).all()) and torch.equal(got[:, 1, 77], o[:, 1, 77])
    fine = torch.isfinite(o)
    assert int(fine.sum()) == n * (256 - 1)
    assert bool(((got - o).abs() <= bo)[fine].all())


@pytest.mark.parametrize("delta", [True, False])
def test_tree_decays_above_one(ext, D, dev, delta):
    q, k, v, gate, beta = _lin_case(24, 1, 2, delta, seed=8)
    gate[::3] = 0.7
    g = torch.Generator().manual_seed(8)
    parents, ptr, slot = _parents([24], "near", g), _ptr([24]), torch.zeros(1, dtype=I32)
    state = 0.3 * torch.randn(1, 2, 128, 128, generator=g)
    got = ext.linattn_tree(*_put(dev, q, k, v, gate, beta, state, slot, ptr, parents))
    _check_tree(D, (q, k, v, gate, beta), state, slot, ptr, parents, 128 ** -0.5, got)


KEEPS = [
    # rows, kept, HK, G
    ([1], [1], 1, 1), ([3, 0, 5], [2, 0, 5], 2, 3), ([12] * 7, [1, 4, 12, 0, 7, 3, 2], 1, 3), ([70], [66], 1, 1),
]


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("case", range(len(KEEPS)))
def test_keep(ext, D, dev, case, delta):
    lengths, kept, HK, G = KEEPS[case]
    _say(f"case keep {case} delta={delta}")
    g = torch.Generator().manual_seed(case)
    N, B = sum(lengths), len(lengths)
    q, k, v, gate, beta = _lin_case(N, HK, G, delta, seed=case, sharp=case % 2 == 1)
    path = torch.cat([torch.cat([torch.randperm(n, generator=g)[:m].sort()[0], torch.full((n - m,), -1)])
                      for n, m in zip(lengths, kept)]).int()
    state = 0.3 * torch.randn(B + 2, HK * G, 128, 128, generator=g)
    slot = torch.randperm(B + 2, generator=g)[:B].int()
    count, ptr = torch.tensor(kept, dtype=I32), _ptr(lengths)
    d = _put(dev, k, v, gate, beta, state, slot, ptr, path, count)
    assert ext.linattn_keep(*d) is None
    st, bs = D.linattn_keep(k, v, gate, beta, state, slot.tolist(), ptr.tolist(), path, count)
    err = (d[4].cpu().double() - st).abs()
    _say(f"  {(err / bs.clamp_min(1e-300)).max().item():.3f} of the bound")
    assert bool((err <= bs).all())


def test_keep_odd_slots_and_paths(ext, D, dev):
    """Slots named again, idle and outside; counts below nothing and above the rows; entries that are no rows; falling
    pointers. States that no sequence takes forward keep their bits."""
    g = torch.Generator().manual_seed(4)
    lengths = [4] * 8
    q, k, v, gate, beta = _lin_case(34, 1, 2, True, seed=4)
    path = torch.tensor([0, 1, 2, 3] * 8 + [0, 1], dtype=I32)
    path[8:12] = torch.tensor([0, -1, 9, 3])
    path[28:32] = torch.tensor([3, 3, 0, -(1 << 31)])
    count = torch.tensor([2, 3, 4, -5, 100, 0, 1, 4], dtype=I32)
    slot = torch.tensor([3, 3, 0, 1, 5, 2, -1, 4], dtype=I32)
    state = 0.3 * torch.randn(5, 2, 128, 128, generator=g)
    for ptr in (_ptr(lengths), _ptr(lengths, 2), torch.tensor([0, 9, 4, 12, 40, 30, -3, 32, 33], dtype=I32)):
        d = _put(dev, k, v, gate, beta, state, slot, ptr, path, count)
        ext.linattn_keep(*d)
        st, bs = D.linattn_keep(k, v, gate, beta, state, slot.tolist(), ptr.tolist(), path, count)
        got = d[4].cpu()
        assert bool(((got.double() - st).abs() <= bs).all())
        still = (st == state.double()).flatten(1).all(1)
        assert torch.equal(got[still], state[still]) and int(still.sum()) >= 2


def test_keep_is_steps(ext, dev):
    """The kept tokens one by one through linattn_step leave the same states, to fp32's rounding."""
    B, n, HV = 3, 6, 6
    q, k, v, gate, beta = _put(dev, *_lin_case(B * n, 2, 3, True, seed=11))
    state = 0.3 * torch.randn(B, HV, 128, 128, device=dev)
    other, slot = state.clone(), torch.tensor([2, 0, 1], dtype=I32, device=dev)
    path = torch.tensor([0, 2, 3, 5, -1, -1] * B, dtype=I32, device=dev)
    ext.linattn_keep(k, v, gate, beta, state, slot, torch.arange(0, 19, 6, dtype=I32, device=dev), path,
                     torch.full((B,), 4, dtype=I32, device=dev))
    outs = []
    for i in (0, 2, 3, 5):
        at = torch.arange(B, device=dev) * n + i
        outs.append(ext.linattn_step(q[at], k[at], v[at], gate[at], beta[at], other, slot))
    assert bool(((state - other).norm(dim=(2, 3)) <= 1e-6 * other.norm(dim=(2, 3))).all())
    # and a tree's outputs along a path are those of the steps
    parents = torch.tensor([-1, 0, 0, 2, 1, 3] * B, dtype=I32, device=dev)
    start = 0.3 * torch.randn(B, HV, 128, 128, device=dev)
    o = ext.linattn_tree(q, k, v, gate, beta, start, slot, torch.arange(0, 19, 6, dtype=I32, device=dev), parents)
    for i in (0, 2, 3, 5):
        at = torch.arange(B, device=dev) * n + i
        want = ext.linattn_step(q[at], k[at], v[at], gate[at], beta[at], start, slot)
        assert bool(((o[at].float() - want.float()).abs() <= 2 * 2.0 ** -8 * want.float().abs() + 1e-4).all())


def test_lintree_past_32_bits(ext, D, dev):
    """States whose byte offsets pass 2^32."""
    HV, slots = 48, 1500
    state = torch.zeros(slots, HV, 128, 128, device=dev)
    q, k, v, gate, beta = _lin_case(3, 16, 3, True, seed=12)
    small = 0.3 * torch.randn(1, HV, 128, 128, generator=torch.Generator().manual_seed(1))
    state[slots - 1].copy_(small[0])
    slot, ptr = torch.tensor([slots - 1], dtype=I32), _ptr([3])
    got = ext.linattn_tree(*_put(dev, q, k, v, gate, beta), state, *_put(dev, slot, ptr))
    _check_tree(D, (q, k, v, gate, beta), small, torch.zeros(1, dtype=I32), ptr, None, 128 ** -0.5, got)
    path, count = torch.arange(3, dtype=I32), torch.tensor([3], dtype=I32)
    ext.linattn_keep(*_put(dev, k, v, gate, beta), state, *_put(dev, slot, ptr, path, count))
    st, bs = D.linattn_keep(k, v, gate, beta, small, [0], ptr.tolist(), path, count)
    assert bool(((state[slots - 1].cpu().double() - st[0]).abs() <= bs[0]).all())
    assert not bool(state[:slots - 1].any())


def test_lintree_empty(ext, dev):
    e = lambda *s, t=BF16: torch.empty(*s, dtype=t, device=dev)  # noqa: E731
    z = lambda *s: torch.zeros(*s, dtype=I32, device=dev)  # noqa: E731
    st = torch.randn(2, 2, 128, 128, device=dev)
    keep = st.clone()
    assert ext.linattn_tree(e(0, 128), e(0, 128), e(0, 256), e(0, 2, t=F32), None, st, z(2), z(3)).shape == (0, 256)
    ext.linattn_keep(e(0, 128), e(0, 256), e(0, 2, t=F32), None, st, z(2), z(3), z(0), z(2))
    x, v, g = torch.ones(3, 128, dtype=BF16, device=dev), torch.ones(3, 256, dtype=BF16, device=dev), torch.zeros(3, 2, device=dev)
    assert not bool(ext.linattn_tree(x, x, v, g, None, st, z(0), z(1)).any())          # rows, and no sequence
    none = e(0, 2, 128, 128, t=F32)
    assert bool(torch.isnan(ext.linattn_tree(x, x, v, g, None, none, z(1), torch.tensor([0, 3], dtype=I32, device=dev))).all())
    ext.linattn_keep(x, v, g, None, none, z(1), torch.tensor([0, 3], dtype=I32, device=dev), z(3), z(1) + 1)
    assert torch.equal(st, keep)


# ---------------------------------------------------------------------------------------------------------------- cache
def _pool(layers, pages, HKV, page, D, fmt, seed, dev):
    g = torch.Generator(device=dev).manual_seed(seed)
    shape = (layers, pages, HKV, page, D)
    kv = [torch.randint(-(1 << 15), 1 << 15, shape, generator=g, device=dev, dtype=torch.int16).view(BF16) if fmt == "bf16" else
          torch.randint(0, 256, shape, generator=g, device=dev, dtype=torch.uint8).view(torch.float8_e4m3fn) for _ in range(2)]
    sc = [torch.rand(shape[:4], generator=g, device=dev) if fmt == "e4m3" else None for _ in range(2)]
    return kv + sc


def _raw(t):
    return t.view({2: torch.int16, 1: torch.uint8, 4: torch.int32}[t.element_size()])


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("lengths,ctx,HKV,D_,page,layers", [
    ([1], [0], 1, 128, 16, 1), ([6], [13], 4, 256, 16, 1), ([12, 0, 5, 9], [250, 3, 0, 64], 2, 256, 32, 3),
    ([70, 33], [40, 1], 1, 128, 64, 2), ([150], [7], 3, 256, 1008, 1), ([8] * 20, list(range(20)), 2, 128, 16, 16)])
def test_keep_rows(ext, D, dev, lengths, ctx, HKV, D_, page, layers, fmt):
    _say(f"case rows {lengths} page={page} layers={layers} {fmt}")
    g = torch.Generator().manual_seed(page)
    need = [-(-(x + y) // page) for x, y in zip(lengths, ctx)]
    pages = sum(need) + 2
    order, at = torch.randperm(pages, generator=g).int(), 0
    table = torch.full((len(lengths), max(need) + 1), -1, dtype=I32)
    for b in range(len(lengths)):
        table[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
    kept = [min(n, 1 + int(torch.randint(0, n + 1, (1,), generator=g))) if n else 0 for n in lengths]
    path = torch.cat([torch.cat([torch.randperm(n, generator=g)[:m].sort()[0], torch.full((n - m,), -1)])
                      for n, m in zip(lengths, kept)]).int()
    cache = _pool(layers, pages, HKV, page, D_, fmt, 1, dev)
    want = [_raw(t).cpu().clone() for t in cache if t is not None]
    count, ptr, c = torch.tensor(kept, dtype=I32), _ptr(lengths), torch.tensor(ctx, dtype=I32)
    D.keep_rows(want, table, ctx, ptr.tolist(), path, kept, page)
    flat = cache if layers > 1 else [None if t is None else t[0] for t in cache]          # one layer: without its axis
    assert ext.kv_cache_keep(*flat[:2], *_put(dev, table, c, ptr, path, count), *flat[2:]) is None
    for t, w in zip([t for t in cache if t is not None], want):
        assert torch.equal(_raw(t).cpu(), w)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
def test_keep_rows_odd(ext, D, dev, fmt):
    """Pages outside the cache, tables that end early, paths that do not rise, counts and pointers that are none."""
    page, HKV, pages = 16, 2, 12
    lengths = [40, 20, 6, 6, 6]
    g = torch.Generator().manual_seed(2)
    table = torch.randperm(pages, generator=g)[:10].int().reshape(5, 2)
    table[1, 1], table[2, 0], table[3, 1] = -7, pages, 1 << 30
    ctx = torch.tensor([5, 10, 12, 14, -3], dtype=I32)
    path = torch.cat([torch.arange(0, 80, 2)[:40] % 40, torch.arange(20).flip(0), torch.tensor([0, 5, 5, 2, -1, 99]),
                      torch.tensor([1, 2, 3, 4, 5, 6]), torch.tensor([5, 4, 3, 2, 1, 0]), torch.tensor([3, 3])]).int()
    count = torch.tensor([40, 20, 6, 6, 1000], dtype=I32)
    for ptr in (_ptr(lengths), torch.tensor([0, 50, 44, 70, 90, 3], dtype=I32)):
        cache = _pool(2, pages, HKV, page, 256, fmt, 3, dev)
        want = [_raw(t).cpu().clone() for t in cache if t is not None]
        D.keep_rows(want, table, ctx, ptr.tolist(), path, count, page)
        ext.kv_cache_keep(*cache[:2], *_put(dev, table, ctx, ptr, path, count), *cache[2:])
        for t, w in zip([t for t in cache if t is not None], want):
            assert torch.equal(_raw(t).cpu(), w)


def _page_lists(table, ctx, refs):
    return table.tolist(), ctx.tolist(), refs.tolist()


@pytest.mark.parametrize("B,MP,pages,page", [(1, 1, 1, 16), (3, 4, 9, 16), (8, 7, 40, 32), (70, 5, 300, 64),
                                             (5, 700, 4500, 16), (1100, 3, 2000, 16), (4, 6, 0, 16), (6, 0, 5, 16)])
def test_pages_over_a_life(ext, D, dev, B, MP, pages, page):
    """Resizes and forks one after the other, beams that change places and pools that run out among them, against lists."""
    _say(f"case pages B={B} MP={MP} pages={pages}")
    g = torch.Generator().manual_seed(B + MP)
    rnd = lambda lo, hi: int(torch.randint(lo, hi, (1,), generator=g))  # noqa: E731
    table, ctx = torch.full((B, MP), -1, dtype=I32), torch.zeros(B, dtype=I32)
    refs = (torch.rand(pages, generator=g) < 0.1).int()                     # held elsewhere
    d = _put(dev, table, ctx, refs)
    T, L, R = _page_lists(table, ctx, refs)
    for turn in range(12):
        if turn % 3 != 2:
            full = MP * page
            tokens = [rnd(-1, max(1, min(full, 3 * full // (1 + turn % 4)) + 1)) for _ in range(B)]
            if turn == 4:
                tokens[0] = (1 << 31) - 1
            if turn == 7:
                tokens = [0] * B
            miss = ext.kv_pages_resize(d[0], d[2], torch.tensor(tokens, dtype=I32).to(dev), page)
            assert miss.tolist() == D.resize(T, R, tokens, page)
            new = [min(max(0, t if t >= 0 else L[b]), full) for b, t in enumerate(tokens)]
            L = new
            d[1].copy_(torch.tensor(L, dtype=I32))
        else:
            src = [rnd(0, B) if rnd(0, 3) else b for b in range(B)]
            if turn == 5:
                src[0], src[-1] = -1, B
            if turn == 8:
                src = list(range(1, B)) + [0]
            pairs = ext.kv_pages_fork(d[0], d[1], d[2], torch.tensor(src, dtype=I32).to(dev), page)
            assert pairs.tolist() == [list(x) for x in D.fork(T, L, R, src, page)]
            assert d[1].tolist() == L
        assert d[0].tolist() == T, turn
        assert d[2].tolist() == R, turn


def test_pages_in_a_large_pool(ext, D, dev):
    """Free pages that lie far apart, and at the very end of the pool."""
    pages, B, MP = 300001, 9, 40
    refs = torch.ones(pages, dtype=I32)
    free = torch.tensor([3, 4095, 4096, 5000, 99999, 262143, 299999, 300000])
    refs[free] = torch.tensor([0, -1, 0, 0, -5, 0, 0, 0], dtype=I32)
    table = torch.full((B, MP), -1, dtype=I32)
    d = _put(dev, table, refs)
    tokens = [16, 0, 40, -1, 16, 0, 17, 32, 16]
    T, R = table.tolist(), refs.tolist()
    miss = ext.kv_pages_resize(d[0], d[1], torch.tensor(tokens, dtype=I32).to(dev), 16)
    assert miss.tolist() == D.resize(T, R, tokens, 16) and sum(miss.tolist()) == 2
    assert d[0].tolist() == T and d[1].tolist() == R


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("HKV,page,D_,layers", [(1, 16, 128, 1), (4, 64, 256, 3), (3, 48, 128, 2)])
def test_pages_copy(ext, dev, HKV, page, D_, layers, fmt):
    pages = 13
    cache = _pool(layers, pages, HKV, page, D_, fmt, 5, dev)
    want = [_raw(t).clone() for t in cache if t is not None]
    pairs = torch.tensor([[0, 7], [-1, 3], [12, 8], [0, 9], [4, -1], [4, 13], [1 << 30, 2], [5, 5], [11, 10]], dtype=I32)
    for a, b in ((0, 7), (12, 8), (0, 9), (11, 10)):
        for w in want:
            w[:, b] = w[:, a]
    flat = cache if layers > 1 else [None if t is None else t[0] for t in cache]
    assert ext.kv_pages_copy(*flat[:2], pairs.to(dev), *flat[2:]) is None
    for t, w in zip([t for t in cache if t is not None], want):
        assert torch.equal(_raw(t), w)


def test_cache_moves_past_32_bits(ext, dev):
    """Rows and pages whose byte offsets pass 2^32, in one layer and over several."""
    HKV, D_, page, pages = 4, 256, 64, 20000
    kc = torch.zeros(2, pages, HKV, page, D_, dtype=BF16, device=dev)
    vc = torch.zeros_like(kc)
    kc[:, pages - 1, :, 3], vc[:, pages - 1, :, 3] = 5.0, 6.0
    z = lambda *x: torch.tensor(x, dtype=I32, device=dev)  # noqa: E731
    ext.kv_pages_copy(kc, vc, z(pages - 1, pages - 2).reshape(1, 2))
    assert bool((kc[:, pages - 2, :, 3] == 5).all()) and bool((vc[:, pages - 2, :, 3] == 6).all())
    ext.kv_cache_keep(kc, vc, z(pages - 1).reshape(1, 1), z(1), z(0, 4), z(0, 2, -1, -1), z(2))
    assert bool((kc[:, pages - 1, :, 2] == 5).all()) and bool((vc[:, pages - 1, :, 2] == 6).all())
    assert int(kc.count_nonzero()) == int(vc.count_nonzero()) == 3 * 2 * HKV * D_


def test_cache_moves_empty(ext, dev):
    z = lambda *s: torch.zeros(*s, dtype=I32, device=dev)  # noqa: E731
    kc = torch.ones(3, 2, 16, 128, dtype=BF16, device=dev)
    keep = kc.clone()
    ext.kv_cache_keep(kc, kc, z(0, 2), z(0), z(1), z(5), z(0))
    ext.kv_cache_keep(kc, kc, z(2, 0), z(2), z(3), z(0), z(2))
    ext.kv_cache_keep(kc[:0], kc[:0], z(1, 2), z(1), torch.tensor([0, 2], dtype=I32, device=dev), z(2), z(1) + 2)
    ext.kv_pages_copy(kc, kc, z(0, 2))
    ext.kv_pages_copy(kc[:0], kc[:0], z(3, 2))
    assert torch.equal(kc, keep)
    assert ext.kv_pages_resize(z(0, 3), z(4), z(0), 16).shape == (0,)
    assert ext.kv_pages_fork(z(0, 3), z(0), z(4), z(0), 16).shape == (0, 2)


# ---------------------------------------------------------------------------------------------------- as they are used
def _server(ext, dev, seed):
    """A drafted step of a small hybrid model on buffers that stay: one full- and one linear-attention layer, logits,
    verification, and the caches taken forward. Returns the step, what it reads, and what it leaves."""
    g = torch.Generator(device=dev).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    B, n, HQ, HKV, D_, page, MP, V, HV = 3, 5, 6, 2, 256, 16, 8, 304, 3
    N, pages = B * n, B * MP
    kc, vc = rn(pages, HKV, page, D_).bfloat16(), rn(pages, HKV, page, D_).bfloat16()
    s = dict(table=torch.full((B, MP), -1, dtype=I32, device=dev), refs=torch.zeros(pages, dtype=I32, device=dev),
             ctx=torch.tensor([13, 30, 47], dtype=I32, device=dev), kc=kc, vc=vc, state=0.1 * rn(B, HV, 128, 128),
             q_ptr=torch.arange(0, N + 1, n, dtype=I32, device=dev), q=rn(HQ, N, D_).bfloat16(), kt=rn(HKV, N, D_).bfloat16(),
             vt=rn(HKV, N, D_).bfloat16(), parents=torch.tensor([-1, 0, 0, 1, 3] * B, dtype=I32, device=dev),
             tokens=torch.randint(0, V, (N,), generator=g, device=dev), u=torch.rand(N, generator=g, device=dev),
             slot=torch.tensor([2, 0, 1], dtype=I32, device=dev), w=(rn(V, HQ * D_) * 0.05).bfloat16(),
             src=torch.tensor([0, 0, 2], dtype=I32, device=dev))
    lin = _put(dev, *_lin_case(N, 1, 3, True, seed))
    bits = ext.tree_bits([[-1, 0, 0, 1, 3]] * B).to(dev)
    probs = torch.softmax(rn(N, V), -1)
    j = torch.arange(n, device=dev)
    ext.kv_pages_resize(s["table"], s["refs"], s["ctx"], page)

    def step():
        missing = ext.kv_pages_resize(s["table"], s["refs"], s["ctx"] + n, page)
        pos = (s["ctx"][:, None] + j).long()
        slots = (torch.gather(s["table"], 1, pos // page).long() * page + pos % page).reshape(-1)
        ext.kv_cache_write(s["kt"], s["vt"], slots, kc, vc)
        y = ext.tree_attn(s["q"], kc, vc, s["table"], s["ctx"], s["q_ptr"], bits)
        o = ext.linattn_tree(*lin, s["state"], s["slot"], s["q_ptr"], s["parents"])
        logits = ext.mm(y, s["w"])[:, :V - 3]
        path, count, nxt = ext.verify_drafts(logits, s["tokens"], s["q_ptr"], s["u"], s["parents"], probs[:, :V - 3])
        ext.kv_cache_keep(kc, vc, s["table"], s["ctx"], s["q_ptr"], path, count)
        ext.linattn_keep(*lin[1:], s["state"], s["slot"], s["q_ptr"], path, count)
        s["ctx"].add_(count)
        ext.kv_pages_resize(s["table"], s["refs"], s["ctx"], page)
        pairs = ext.kv_pages_fork(s["table"], s["ctx"], s["refs"], s["src"], page)
        ext.kv_pages_copy(kc, vc, pairs)
        return [y, o, logits, path, count, nxt, missing, pairs]

    return step, s, lin, bits, probs


def test_step_runs_together(ext, D, dev):
    """Every operator of a drafted step against the oracle on what the one before gave."""
    from oracle import cores_oracle as C
    step, s, lin, bits, probs = _server(ext, dev, 3)
    before = {k: t.cpu().clone() for k, t in s.items()}
    y, o, logits, path, count, nxt, missing, pairs = step()
    torch.cuda.synchronize()
    cpu = lambda t: t.cpu()  # noqa: E731
    assert missing.tolist() == [0] * 3
    T, R, L = before["table"].tolist(), before["refs"].tolist(), before["ctx"].tolist()
    D.resize(T, R, [x + 5 for x in L], 16)
    kc, vc = before["kc"], before["vc"]
    for b in range(3):
        for j in range(5):
            pos = L[b] + j
            kc[T[b][pos // 16], :, pos % 16], vc[T[b][pos // 16], :, pos % 16] = (before[x][:, 5 * b + j] for x in ("kt", "vt"))
    table = torch.tensor(T, dtype=I32)
    want, _, bo, _ = C.tree_attn(before["q"], kc, vc, None, None, table, before["ctx"], before["q_ptr"], bits.cpu(), 1 / 16)
    assert bool(((cpu(y).double().reshape(want.shape) - want).abs() <= bo).all())
    args = [cpu(t) for t in lin]
    _check_tree(D, args, before["state"], before["slot"], before["q_ptr"], before["parents"], 128 ** -0.5, o)
    c = dict(logits=cpu(logits), tokens=before["tokens"], q_ptr=before["q_ptr"], u=before["u"], parents=before["parents"],
             probs=cpu(probs)[:, :301], temperature=None)
    _check_verify(D, c, [cpu(path), cpu(count), cpu(nxt)])
    caches = [_raw(kc[None]).clone(), _raw(vc[None]).clone()]
    D.keep_rows(caches, table, L, before["q_ptr"].tolist(), cpu(path), count.tolist(), 16)
    st, bs = D.linattn_keep(*args[1:], before["state"], before["slot"].tolist(), before["q_ptr"].tolist(), cpu(path), cpu(count))
    assert bool(((cpu(s["state"]).double() - st).abs() <= bs).all())
    L = [x + m for x, m in zip(L, count.tolist())]
    D.resize(T, R, L, 16)
    pairs_want = D.fork(T, L, R, before["src"].tolist(), 16)
    assert cpu(pairs).tolist() == [list(x) for x in pairs_want]
    for a, b in pairs_want:
        if a >= 0 and b >= 0:
            for x in caches:
                x[:, b] = x[:, a]
    assert s["table"].tolist() == T and s["refs"].tolist() == R and s["ctx"].tolist() == L
    assert torch.equal(_raw(s["kc"]).cpu(), caches[0][0]) and torch.equal(_raw(s["vc"]).cpu(), caches[1][0])


def test_steps_in_two_graphs(ext, dev):
    """Two servers' captured steps, replayed in turn with eager work between, go the way of eager steps: states, contexts and
    tables move on with every replay."""
    runs = []
    for seed in (5, 6):
        step, s, *_ = _server(ext, dev, seed)
        start = {k: t.clone() for k, t in s.items()}

        def reset(s=s, start=start):
            for k, t in s.items():
                t.copy_(start[k])

        want = []
        for r in range(3):
            outs = [x.clone() for x in step()]
            want.append((outs, {k: t.clone() for k, t in s.items()}))
        reset()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.synchronize()
        reset()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = step()
        runs.append((graph, outs, want, s, reset, step))        # the step holds what its graph reads
    for _ in range(2):
        for run in runs:
            run[4]()
        for r in range(3):
            for graph, outs, want, s, *_ in runs:
                graph.replay()
                torch.cuda.synchronize()
                for i, (a, b) in enumerate(zip(outs, want[r][0])):
                    assert torch.equal(a, b), f"replay {r}: output {i}"
                for k, t in s.items():
                    assert torch.equal(t, want[r][1][k]), f"replay {r}: {k}"
                torch.randn(1 << 20, device=dev).sum().item()              # eager work that takes memory
            _server(ext, dev, 9)[0]()


def test_steps_on_streams_at_once(ext, dev):
    lots = []
    for seed in (7, 8):
        step, s, *_ = _server(ext, dev, seed)
        start = {k: t.clone() for k, t in s.items()}
        want = [x.clone() for x in step()]
        for k, t in s.items():
            t.copy_(start[k])
        lots.append((step, want, torch.cuda.Stream()))
    torch.cuda.synchronize()
    got = []
    for step, want, side in lots:
        with torch.cuda.stream(side):
            got.append(step())
    torch.cuda.synchronize()
    for (step, want, side), outs in zip(lots, got):
        for i, (a, b) in enumerate(zip(outs, want)):
            assert torch.equal(a, b), f"output {i}"


def test_verify_no_rows_in_c(pkg, dev):
    """A step without rows, with draft probabilities of a large vocabulary, as a host in C may call it: counts of 0, no next
    tokens, and a workspace of no bytes."""
    L = pkg._lib.lib()
    ptr, some = torch.zeros(4, dtype=I32, device=dev), torch.ones(16, device=dev)
    for parents in (None, ptr.data_ptr()):
        for V in (10, 41000, 1 << 22):
            count, nxt = torch.full((3,), 77, dtype=I32, device=dev), torch.full((3,), 77, device=dev)
            assert L.ojx_verify_drafts_workspace(0, 3, V, 1) == 0
            assert L.ojx_verify_drafts(None, 0, V, None, ptr.data_ptr(), None, parents, some.data_ptr(), 0, V, None, 0, 3, V,
                                       None, count.data_ptr(), nxt.data_ptr(), None, 0, None) == 0
            torch.cuda.synchronize()
            assert count.tolist() == [0] * 3 and nxt.tolist() == [-1] * 3, V


def _near_borders(T, least, most, count):
    """Logits x (beside one of 0) and numbers u, all fp32, with u between `least` and `most` from e^(x/T) / (1 + e^(x/T)) or from
    the other's share, relative to them: (x, u, below) of each kind. In 80 bits, whose exponential is off by some 1e-19."""
    import numpy as np
    x = np.linspace(-12.0, -1e-3, 1 << 22).astype(np.float32)
    e = np.exp(x.astype(np.longdouble) / np.longdouble(np.float32(T)))
    out = []
    for p in (e / (1 + e), 1 / (1 + e)):
        u = p.astype(np.float32)
        off = u.astype(np.longdouble) / p - 1
        at = np.nonzero((np.abs(off) > least) & (np.abs(off) < most))[0][:count]
        assert len(at) >= min(count, 20)
        out.append((torch.from_numpy(x[at]), torch.from_numpy(u[at]), (off[at] < 0).tolist()))
    return out


@pytest.mark.parametrize("T", [1.0, 0.7])
@pytest.mark.parametrize("V,probs", [(2, False), (2, True), (9000, True), (41000, False), (41000, True)])
def test_verify_decides_in_64_bits(ext, dev, V, probs, T):
    """Numbers 2e-14 to 1e-12 beside the border of a test and of a draw, a distance that 64 bits tell and fewer do not. A
    probability is off by the argument's roundings, four times 2^-53 of |x / T| <= 17.2, by the exponential's 3.2e-16 and its
    rounding, 2^-52, and by those of a sum and quotient of two such: 2 (4 17.2 2^-53 + 3.2e-16 + 2^-52) + 4 2^-53 < 1.8e-14."""
    test, draw = _near_borders(T, 2e-14, 1e-12, 60)
    ends = (0, V - 1)
    for kind, (x, u, below) in (("test", test), ("draw", draw)):
        B, n = len(x), 2 if kind == "test" else 1
        logits = torch.full((B * n, V), -math.inf)
        logits[:, ends[0]] = 0.0
        logits[:, ends[1]] = x.repeat_interleave(n)
        q = torch.zeros(B * n, V)
        q[:, ends[1]] = 1.0
        tokens = torch.full((B * n,), ends[1])
        numbers = u if kind == "draw" else torch.stack([torch.full_like(u, 0.5), u], 1).reshape(-1)
        for tree in (None, torch.tensor([-1, 0][:n] * B, dtype=I32)):
            got = _run_verify(ext, {"logits": logits, "tokens": tokens, "q_ptr": torch.arange(0, B * n + 1, n, dtype=I32),
                                    "u": numbers, "parents": tree, "probs": q if probs else None,
                                    "temperature": torch.full((B,), T)}, dev)
            if kind == "test":
                assert got[1].tolist() == [1 + b for b in below]
            else:
                assert got[2].tolist() == [ends[0] if b else ends[1] for b in below]


@pytest.mark.parametrize("V", [7, 9000, 41000])
def test_verify_little_left_without_probabilities(ext, D, dev, V):
    """Looked-up tokens that are nearly certain, rejected one after the other: each time some e^-16 of what was there is left,
    which one less their shares does not give. Then tokens that share the rest alike, tested on both sides of their share."""
    g = torch.Generator().manual_seed(V)
    up = 1.0 - 2.0 ** -24
    lots = []
    for B in range(24):
        deep = 1 + B % 3
        at = torch.randperm(V, generator=g)[:deep + 4].tolist()
        x = torch.full((V,), -math.inf)
        for i, a in enumerate(at):
            x[a] = -16.0 * min(i, deep) + (0.0 if i < deep else 0.1 * (i - deep))
        share = torch.softmax(x[at[deep:]].double(), 0)
        first = float(share[0])
        u = (first * 0.999, first * 1.001)[B // 3 % 2]
        second = float(share[1]) / (1.0 - first)
        lots.append((x, [at[0]] + at[:deep] + at[deep:deep + 2], [0.4] + [up] * deep + [u, second * (0.999, 1.001)[B // 6 % 2]]))
    n = [len(t) for _, t, _ in lots]
    c = {"logits": torch.cat([x.repeat(k, 1) for (x, _, _), k in zip(lots, n)]),
         "tokens": torch.tensor([t for _, ts, _ in lots for t in ts]), "q_ptr": _ptr(n),
         "u": torch.tensor([t for _, _, us in lots for t in us], dtype=F32),
         "parents": torch.tensor([j for k in n for j in [-1] + [0] * (k - 1)], dtype=I32), "probs": None, "temperature": None}
    count = _check_verify(D, c, _run_verify(ext, c, dev), least=1e-9)
    assert set(count) == {1, 2}


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("n", [1, 20, 64, 100, 300])
def test_tree_states_in_fp32(ext, D, dev, n, delta):
    """States enter as exactly as fp32 products take them: keys and queries that read the difference of two key dims which agree
    to 13 bits. Every row follows the state. With the delta rule a row's query reads its own key alone, so that its output is
    -(x - y) of its key, otherwise x - y of its query. Bound: a sum of six pieces' products, each off by two fp32 roundings of
    the magnitudes, and the output's rounding to bf16, beside which four fp32 roundings of the output."""
    g = torch.Generator().manual_seed(n)
    HV = 2
    state = torch.randn(1, HV, 128, 128, generator=g)
    state[:, :, 1:126:3] = state[:, :, 0:126:3] * (1 + 2.0 ** -13 * torch.randn(1, HV, 42, 128, generator=g))
    state[:, :, 2:126:3] = 0.0
    i = torch.arange(n)
    x = 3 * (i % 42)
    pick = torch.zeros(n, 128)
    pick[i, x], pick[i, x + 1] = 1.0, -1.0
    q, k = pick.clone(), torch.zeros(n, 128)
    if delta:
        q, k = torch.zeros(n, 128), pick.clone()
        q[i, x + 2] = k[i, x + 2] = 1.0
    args = (q.bfloat16(), k.bfloat16(), torch.zeros(n, HV * 128, dtype=BF16), torch.zeros(n, HV),
            torch.ones(n, HV, dtype=BF16) if delta else None)
    parents, slot, ptr = torch.full((n,), -1, dtype=I32), torch.zeros(1, dtype=I32), _ptr([n])
    o = D.linattn_tree(*args, state, [0], [0, n], parents, 1.0)[0]
    got = ext.linattn_tree(*_put(dev, *args, state, slot, ptr, parents), scale=1.0).cpu().double().reshape(o.shape)
    a, b = state[0][:, x].double().abs().transpose(0, 1), state[0][:, x + 1].double().abs().transpose(0, 1)
    bound = 12 * 2.0 ** -24 * (a + b) + (2.0 ** -8 + 4 * 2.0 ** -24) * o.abs()
    _say(f"  out {((got - o).abs() / bound).max().item():.3f} of its bound")
    assert bool(((got - o).abs() <= bound).all())


def _bits(t):
    return _raw(t.contiguous()).cpu()


@pytest.mark.parametrize("delta", [True, False])
def test_tree_repeats_itself(ext, dev, delta):
    """Two calls give the same bits, NaN among them: short and long sequences, heads that go row by row after their outputs were
    stored once, sequences whose state is not there."""
    g = torch.Generator().manual_seed(16)
    lengths = [70, 3, 0, 130, 64, 90, 256, 300, 12, 64]
    N, B = sum(lengths), len(lengths)
    q, k, v, gate, beta = _lin_case(N, 1, 3, delta, seed=16)
    parents, ptr = _parents(lengths, "near", g), _ptr(lengths)
    v[int(ptr[3]) + 70, 5], v[int(ptr[4]) + 1, 130] = math.inf, math.nan
    gate[int(ptr[9]) + 2, 1], gate[int(ptr[8]), 0] = 0.5, math.nan
    state = 0.3 * torch.randn(4, 3, 128, 128, generator=g)
    state[3, 2, 4, 4] = math.inf
    slot = torch.tensor([1, -1, 0, 0, 2, 7, 2, 1, 3, 3], dtype=I32)
    d = _put(dev, q, k, v, gate, beta, state, slot, ptr, parents)
    first = _bits(ext.linattn_tree(*d))
    assert int((first != 0).sum()) > 0
    for i in range(20):
        other = torch.full((1 << 22,), i + 0.5, device=dev)      # the workspace's former contents differ from call to call
        del other
        assert torch.equal(_bits(ext.linattn_tree(*d)), first), i


# ------------------------------------------------- verification with launches of their own for the first rejections' sums
def _has_walks(pkg, V):
    """Whether calls with draft probabilities of V tokens have such launches: their workspace holds the walks then."""
    size = pkg._lib.lib().ojx_verify_drafts_workspace
    return size(8, 2, V, 1) > size(8, 2, V, 0)


@pytest.mark.parametrize("kind", ["line", "near", "star", "wide"])
@pytest.mark.parametrize("probs", ["bf16", "fp32"])
@pytest.mark.parametrize("dtype,V,pad", [(BF16, 32761, 0), (BF16, 32762, 3), (F32, 32762, 0), (BF16, 41000, 0), (F32, 41003, 5),
                                         (BF16, 65539, 1)])
def test_verify_walks(ext, pkg, D, dev, dtype, V, pad, probs, kind):
    """Vocabularies around the smallest with such launches and above, rows of any alignment, greedy sequences and empty ones
    among others."""
    assert _has_walks(pkg, V) == (V > 32761)
    _say(f"case walks {V} {dtype} probs={probs} {kind}")
    c = _verify_case([6, 0, 9, 1, 5, 12, 4], V, dtype, probs, kind, pad, seed=V + len(kind), near=1.5)
    _say(f"  accepted {_check_verify(D, c, _run_verify(ext, c, dev))}")


def _rejections(V, patterns, dtype, seed):
    """Sequences in which the first pattern[0] children of row 0 are rejected, then one is accepted, the first pattern[1] of its
    own are, and so on; behind the last ones nothing is accepted. The drafts' distributions are on the even tokens but for one in
    a hundred, the target's on the odd ones but for one in a thousand."""
    g = torch.Generator().manual_seed(seed)
    n = [1 + sum(p) + len(p) - 1 for p in patterns]
    N = sum(n)
    raw = 2.0 * torch.randn(N, V, generator=g)
    odd = (torch.arange(V) % 2).bool()

    def half(mask, weight):
        e = torch.exp(raw) * mask
        return weight * e / e.sum(-1, keepdim=True)

    p = half(odd, 0.999) + half(~odd, 0.001)
    raw = 2.0 * torch.randn(N, V, generator=g)
    q = half(~odd, 0.99) + half(odd, 0.01)
    tokens, parents, u = [], [], []
    for b, pattern in enumerate(patterns):
        at, cur, j = len(tokens), 0, 1
        tokens.append(0), parents.append(-1), u.append(0.1 + 0.8 * float(torch.rand(1, generator=g)))
        for i, k in enumerate(pattern):
            for r in range(k + (i + 1 < len(pattern))):
                here = q[at + cur] * ~odd if r < k else p[at + cur] * odd
                tokens.append(int(torch.multinomial(here, 1, generator=g)))
                parents.append(cur)
                # rejected: q of the even tokens is hundreds of times p; accepted: p of the odd ones hundreds of times q
                u.append(0.9 if r < k else 0.1)
            j += k + 1
            cur = j - 1
    return {"logits": torch.log(p).to(dtype), "tokens": torch.tensor(tokens), "q_ptr": _ptr(n), "u": torch.tensor(u),
            "parents": torch.tensor(parents, dtype=I32), "probs": q, "temperature": None}


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", [9000, 33000, 70001])
def test_verify_counted_rejections(ext, pkg, D, dev, V, dtype):
    """One to dozens of rejections, accepted rows before, between and behind them, so that walks are handed on at every number
    of rejections and taken up by the last kernel before, at and behind the last launch."""
    assert _has_walks(pkg, V) == (V > 32761)
    patterns = [[k] for k in range(0, 10)] + [[0, k] for k in range(0, 9)] + [[k, 0] for k in range(1, 9)]
    patterns += [[2, 3], [5, 1], [6, 1], [7, 2], [1, 6], [3, 3], [3, 4], [1, 1, 1, 1, 1, 1], [1, 1, 1, 1, 1, 1, 1], [2, 2, 2, 0],
                 [2, 2, 2, 1], [0, 0, 6, 0, 1], [12, 12], [30], [70], [66, 3], [1, 70, 1], [0, 0, 0, 0]]
    c = _rejections(V, patterns, dtype, seed=V)
    count = _check_verify(D, c, _run_verify(ext, c, dev))
    hits = sum(x == len(p) for x, p in zip(count, patterns))
    assert hits >= len(patterns) - 3, (hits, len(patterns))


def test_verify_walks_temperatures(ext, pkg, D, dev):
    assert _has_walks(pkg, 33000)
    temps = [0.0, -1.0, math.nan, math.inf, 1e-3, 1e-40, 50.0, 1.0]
    for kind in ("near", "star", "line"):
        c = _verify_case([7] * 8, 33000, BF16, "fp32", kind, seed=5, temps=temps, near=3.0)
        _check_verify(D, c, _run_verify(ext, c, dev))
    c = _verify_case([7] * 8, 33000, F32, "bf16", "star", seed=6, temps=[0.0] * 8)       # nobody has sums to make
    _check_verify(D, c, _run_verify(ext, c, dev))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_verify_walks_masks(ext, pkg, D, dev, dtype):
    """test_verify_masks in a vocabulary with such launches: masked, lowest, infinite and NaN logits, probabilities that are
    none, tokens and parents that are none."""
    V = 33003
    assert _has_walks(pkg, V)
    low = torch.finfo(dtype).min
    for seed in range(4):
        c = _verify_case([7] * 14, V, dtype, "fp32", "near", seed=seed, temps=[1.0, 0.0, 0.8, 1.5, 1.0, 0.9, 0.0] * 2, near=3.0)
        x, P, q = c["logits"], c["parents"], c["probs"]
        x[0:28, 20000:] = -math.inf
        x[7:14, ::2] = low
        x[14:21, 50:] = low
        x[21 + seed, :] = -math.inf
        x[28 + seed, V - 1] = math.nan
        x[35 + seed, 3] = math.inf
        x[42, :] = -math.inf
        x[49, :] = math.nan
        x[56, :] = low
        x[63:70] = -math.inf
        x[63:70, V - 2] = low
        c["tokens"][70:77] = torch.tensor([0, -1, V, 1 << 40, -(1 << 40), V - 1, 0])
        P[77:84] = torch.tensor([5, 1, 7, -3, 0, 100, 3])
        q[84:91, ::3], q[84:91, 1::3] = -1.0, math.nan
        q[91:98] = 0.0
        _check_verify(D, c, _run_verify(ext, c, dev))


def test_verify_walks_rows_of_no_sequence(ext, pkg, D, dev):
    assert _has_walks(pkg, 33000)
    c = _verify_case([3, 4, 0, 8], 33000, BF16, "fp32", "star", seed=2, lead=2, spare=5, near=4.0)
    _check_verify(D, c, _run_verify(ext, c, dev))
    for ptr in ([9, 2, 5, 5, 12], [-4, 3, 2, 18, 19], [0, 100, 3, 5, 7], [2, 2, 2, 2, 2], [22, 22, 22, 22, 22]):
        c["q_ptr"] = torch.tensor(ptr, dtype=I32)
        _check_verify(D, c, _run_verify(ext, c, dev))


def test_verify_walks_past_32_bits(ext, pkg, D, dev):
    assert _has_walks(pkg, 33000)
    c = _verify_case([6], 33000, BF16, "fp32", "star", seed=6, temps=[0.9], near=4.0)
    want = _run_verify(ext, c, dev)
    _check_verify(D, c, want)
    ld = (1 << 29) + 17
    d = {x: None if t is None else t.to(dev) for x, t in c.items()}
    for name in ("logits", "probs"):
        back = torch.empty(5 * ld + 33000, dtype=d[name].dtype, device=dev)
        far = back.as_strided((6, 33000), (ld, 1))
        far.copy_(d[name])
        d[name] = far
    got = ext.verify_drafts(d["logits"], d["tokens"], d["q_ptr"], d["u"], d["parents"], d["probs"], d["temperature"])
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)


def test_verify_walks_in_graphs_and_on_streams(ext, pkg, D, dev):
    """Two captured calls replayed in turn and at once on two streams, with other numbers each time, and eager work between."""
    V = 40000
    assert _has_walks(pkg, V)
    lots = []
    for seed in (1, 2):
        c = _rejections(V, [[k, 9 - k, 2] for k in range(10)], BF16, seed)
        d = {x: None if t is None else t.to(dev) for x, t in c.items()}
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            ext.verify_drafts(**d)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = ext.verify_drafts(**d)
        lots.append((c, d, graph, out, side))
    for turn in range(4):
        for c, d, *_ in lots:
            g = torch.Generator().manual_seed(turn)
            c["u"] = torch.where(torch.rand(len(c["u"]), generator=g) < 0.5, c["u"], torch.rand(len(c["u"]), generator=g))
            d["u"].copy_(c["u"])
        torch.cuda.synchronize()
        for c, d, graph, out, side in lots:
            with torch.cuda.stream(side):
                graph.replay()
            if turn < 2:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        for c, d, graph, out, side in lots:
            got = [t.cpu() for t in out]
            _check_verify(D, c, got)
            for a, b in zip(got, ext.verify_drafts(**d)):
                assert torch.equal(a, b.cpu())
