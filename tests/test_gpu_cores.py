"""GPU parity of the attention cores and the paged cache (ext.kv_cache_write, kv_cache_read, tree_attn, linattn_prompt,
linattn_step) with the 64-bit oracle, which gives the bounds that the outputs are held to (oracle/cores_oracle.py)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

FMT = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}


def _say(*a):
    print(*a, flush=True)


@pytest.fixture(scope="module")
def C():
    from oracle import cores_oracle
    return cores_oracle


# ---------------------------------------------------------------------------------------------------------------- cache
def _pool(pages, HKV, page, D, fmt, dev, fill=None):
    """An empty cache with recognisable contents."""
    if fmt == "bf16":
        kc = torch.full((pages, HKV, page, D), 3.0 if fill is None else fill, dtype=torch.bfloat16, device=dev)
        return kc, kc.clone() + 1, None, None
    kc = torch.full((pages, HKV, page, D), 0x31, dtype=torch.uint8, device=dev)
    sc = torch.full((pages, HKV, page), 0.5, device=dev)
    return kc.view(torch.float8_e4m3fn), (kc + 1).view(torch.float8_e4m3fn), sc, sc + 1


def _rows(HKV, N, D, seed):
    """k, v with rows of every kind: zeros, one non-zero, infinities and NaN, the largest and the smallest values."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(2, HKV, N, D, generator=g) * torch.exp(3 * torch.randn(2, HKV, N, 1, generator=g))
    x = x.bfloat16()
    flat = x.reshape(-1, D)
    special = [lambda r: r.zero_(), lambda r: r.zero_()[5:6].fill_(1e-38), lambda r: r[3:5].fill_(math.inf),
               lambda r: r[7:8].fill_(math.nan), lambda r: r.mul_(2.0 ** 100), lambda r: r.mul_(2.0 ** -120),
               lambda r: r.fill_(-math.inf), lambda r: r[0:2].copy_(torch.tensor([448.0, 449.0])),
               lambda r: r.copy_((torch.arange(D) * 0.125).bfloat16()), lambda r: r.fill_(3.3895e38)]
    for i, f in enumerate(special):
        if flat.shape[0] > 4 * i + 3:
            f(flat[(4 * i + 3) * 7 % flat.shape[0]])
    return x[0].contiguous(), x[1].contiguous()


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("N,HKV,D,page", [(1, 1, 256, 16), (1, 4, 128, 64), (7, 4, 256, 64), (65, 3, 128, 48),
                                          (64, 4, 256, 16), (531, 2, 256, 128)])
def test_cache_write_and_read(ext, C, dev, fmt, N, HKV, D, page):
    _say(f"case cache {fmt} N={N} HKV={HKV} D={D} page={page}")
    k, v = _rows(HKV, N, D, seed=N + D)
    pages = -(-N // page) + 2
    g = torch.Generator().manual_seed(N)
    slots = torch.randperm(pages * page, generator=g)[:N]
    if N > 6:
        slots[2], slots[3], slots[5] = -1, pages * page, -(1 << 40)      # not written
    cache = _pool(pages, HKV, page, D, fmt, dev)
    before = [None if t is None else t.cpu().clone() for t in cache]
    kd, vd = k.to(dev), v.to(dev)
    ext.kv_cache_write(kd.unsqueeze(0), vd.unsqueeze(0), slots.to(dev), *cache)
    k2, v2 = ext.kv_cache_read(cache[0], cache[1], slots.to(dev), cache[2], cache[3])
    torch.cuda.synchronize()
    inside = (slots >= 0) & (slots < pages * page)
    at = slots[inside]
    for x, got, sc, was, wsc, back in ((k, cache[0], cache[2], before[0], before[2], k2),
                                       (v, cache[1], cache[3], before[1], before[3], v2)):
        x = x[:, inside]
        got = got.cpu()
        if fmt == "bf16":
            want = was.clone()
            want.transpose(1, 2).reshape(pages * page, HKV, D)           # a view check: the index below is the layout
            want[at // page, :, at % page] = x.transpose(0, 1)
            assert torch.equal(got.view(torch.int16), want.view(torch.int16))
            ref = x
        else:
            val, scale = C.cache_store(x)
            raw, wraw = got.view(torch.uint8), was.view(torch.uint8).clone()
            there = C._TABLE[raw.long()][at // page, :, at % page].transpose(0, 1)
            assert torch.equal(torch.nan_to_num(there, nan=999.0), torch.nan_to_num(val, nan=999.0))
            assert torch.equal(sc.cpu()[at // page, :, at % page].transpose(0, 1).double(), scale)
            raw[at // page, :, at % page] = wraw[at // page, :, at % page]
            assert torch.equal(raw, wraw)                                # nothing else was touched
            s = sc.cpu()
            s[at // page, :, at % page] = wsc[at // page, :, at % page]
            assert torch.equal(s, wsc)
            ref = (val * scale[..., None]).float().bfloat16()
        back = back.cpu()
        assert torch.equal(torch.nan_to_num(back[:, inside].float(), nan=999.0), torch.nan_to_num(ref.float(), nan=999.0))
        assert bool((back[:, ~inside] == 0).all())


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
def test_cache_past_32_bits(ext, dev, fmt):
    """Slots whose byte offsets pass 2^32 in a cache of more than 4 GiB."""
    HKV, D, page, pages = 4, 256, 64, 70000 if fmt == "e4m3" else 36000
    kc = torch.zeros(pages, HKV, page, D, dtype=torch.uint8 if fmt == "e4m3" else torch.bfloat16, device=dev)
    vc = torch.zeros_like(kc)
    if fmt == "e4m3":
        kc, vc = kc.view(FMT[fmt]), vc.view(FMT[fmt])
    ks = torch.zeros(pages, HKV, page, device=dev) if fmt == "e4m3" else None
    vs = torch.zeros(pages, HKV, page, device=dev) if fmt == "e4m3" else None
    slots = torch.tensor([5, (pages - 1) * page + 63, (pages // 2) * page + 7], device=dev)
    k = (torch.arange(HKV * 3 * D, device=dev) % 15 - 7).reshape(HKV, 3, D).bfloat16()   # whole numbers: exact in e4m3
    ext.kv_cache_write(k, -k, slots, kc, vc, ks, vs)
    k2, v2 = ext.kv_cache_read(kc, vc, slots, ks, vs)
    assert torch.equal(k2, k) and torch.equal(v2, -k)
    assert torch.equal(kc[pages - 1, :, 63].float() * (ks[pages - 1, :, 63, None] if ks is not None else 1), k[:, 1].float())
    # one sequence whose pages are the last of the cache
    table = torch.tensor([[pages - 1, pages // 2]], dtype=torch.int32, device=dev)
    q = torch.zeros(HKV, 1, D, dtype=torch.bfloat16, device=dev)
    out = ext.tree_attn(q, kc, vc, table, torch.tensor([64 + 7], dtype=torch.int32, device=dev),
                        torch.tensor([0, 1], dtype=torch.int32, device=dev), ks=ks, vs=vs)
    # equal weights over 72 positions, two of them written: the mean of the values
    want = -(k[:, 1].double() + k[:, 2].double()) / 72
    err = (out.reshape(HKV, D).double() - want).abs()
    assert bool((err <= want.abs() * (2.0 ** -8 + 2.0 ** -8) * 1.01 + 15 / 72 * 2.0 ** -8).all())


# ----------------------------------------------------------------------------------------------------------------- tree
def _tree_case(n, ctx, HKV, G, D, page, fmt, dev, seed, words=None, spare=0, chain=False, ext=None):
    """Tensors of a tree-attention call on the CPU and, with the last pages in random order, its cache."""
    g = torch.Generator().manual_seed(seed)
    B, HQ = len(n), HKV * G
    need = [-(-(x + y) // page) for x, y in zip(n, ctx)]
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=g).int()
    table = torch.full((B, max(need) + 1), -1, dtype=torch.int32)
    at = 0
    for b in range(B):
        table[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
    kv = [torch.randn(pages, HKV, page, D, generator=g).bfloat16() for _ in range(2)]
    if fmt == "e4m3":
        sc = [torch.exp2(torch.randint(-4, 1, (pages, HKV, page), generator=g).float()) * 0.7 for _ in range(2)]
        kv = [(x.float() * 2).to(torch.float8_e4m3fn) for x in kv]
    else:
        sc = [None, None]
    N = sum(n) + spare
    q = torch.randn(HQ, N, D, generator=g).bfloat16()
    q_ptr = torch.tensor([0] + list(torch.tensor(n).cumsum(0)), dtype=torch.int32)
    bits = None
    if not chain:
        parents = [[int(torch.randint(-1, j, (1,), generator=g)) for j in range(x)] for x in n]
        bits = ext.tree_bits(parents + [[-1] * spare])
        if words is not None and bits.shape[1] < words:
            bits = torch.cat([bits, torch.zeros(N, words - bits.shape[1], dtype=torch.int64)], 1)
    return {"q": q, "kc": kv[0], "vc": kv[1], "ks": sc[0], "vs": sc[1], "table": table,
            "ctx": torch.tensor(ctx, dtype=torch.int32), "q_ptr": q_ptr, "bits": bits}


def _run_tree(ext, c, dev, scale=None):
    d = {x: None if t is None else t.to(dev) for x, t in c.items()}
    return ext.tree_attn(d["q"], d["kc"], d["vc"], d["table"], d["ctx"], d["q_ptr"], d["bits"], d["ks"], d["vs"],
                         scale=scale, want_lse=True)


def _check_tree(C, c, out, lse, scale):
    HQ, N, D = c["q"].shape
    o, l, bo, bl = C.tree_attn(c["q"], c["kc"], c["vc"], c["ks"], c["vs"], c["table"], c["ctx"], c["q_ptr"], c["bits"],
                               scale)
    got = out.cpu().double().reshape(N, HQ, D)
    assert bool(torch.isfinite(got).all())
    worst = ((got - o).abs() / bo.clamp_min(1e-300)).max().item()
    assert worst <= 1.0, f"out: {worst:.3f} of the bound"
    gl = lse.cpu().double()
    none = torch.isinf(l)
    assert torch.equal(none, gl == -math.inf)
    assert bool(((gl - l).abs()[~none] <= bl[~none]).all())
    _say(f"  out {worst:.3f} of its bound")


TREES = [
    # drafted, cached, HKV, G, D, page
    ([1], [0], 1, 1, 256, 16),
    ([1], [1], 2, 6, 256, 16),
    ([1], [539], 4, 6, 256, 64),
    ([1, 1, 1], [15, 16, 17], 2, 4, 128, 16),
    ([5, 0, 2], [100, 30, 0], 2, 6, 256, 32),
    ([12, 7], [257, 64], 4, 6, 256, 64),
    ([33], [129], 1, 8, 128, 48),
    ([70, 3], [40, 300], 2, 3, 256, 64),
    ([130], [50], 1, 2, 128, 128),
    ([9, 4, 1, 6, 17], [0, 31, 63, 64, 65], 1, 5, 256, 16),
    ([2], [700], 1, 64, 128, 64),
]


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("chain", [False, True])
@pytest.mark.parametrize("case", range(len(TREES)))
def test_tree_attn(ext, C, dev, case, chain, fmt):
    n, ctx, HKV, G, D, page = TREES[case]
    _say(f"case tree {case} {fmt} chain={chain}")
    c = _tree_case(n, ctx, HKV, G, D, page, fmt, dev, seed=case, chain=chain, ext=ext)
    scale = D ** -0.5
    out, lse = _run_tree(ext, c, dev)
    _check_tree(C, c, out, lse, scale)


@pytest.mark.parametrize("scale", [0.0, -0.05, 1.5])
def test_tree_attn_scales(ext, C, dev, scale):
    """No scale, a negative one, and one that leaves a single weight."""
    c = _tree_case([6, 3], [150, 41], 2, 3, 128, 32, "bf16", dev, seed=3, ext=ext)
    out, lse = _run_tree(ext, c, dev, scale)
    _check_tree(C, c, out, lse, scale)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("D", [128, 256])
def test_tree_attn_masks_and_bad_pages(ext, C, dev, D, fmt):
    """Rows that see nothing, rows of no sequence, pages outside the cache, tables that end early; NaN and infinities in
    every place that no row sees, and in drafted tokens that some rows do not see."""
    _say(f"case masks {fmt} D={D}")
    n, ctx, page = [8, 5, 0, 20], [0, 70, 9, 33], 16
    c = _tree_case(n, ctx, 2, 3, D, page, fmt, dev, seed=11, spare=3, ext=ext)
    c["bits"][2] = 0                       # sequence 0 has no context: nothing left
    c["bits"][6] = 1 << 20                 # a bit behind its drafted tokens
    c["table"][1, 1] = -5                  # bad pages in the middle of a context
    c["table"][1, 2] = c["kc"].shape[0] + 3
    c["table"][3, 0] = 1 << 30
    # poison what nobody sees: free pages, places behind a sequence's end
    used = torch.zeros(c["kc"].shape[0], page, dtype=torch.bool)
    for b in range(4):
        for p in range(n[b] + ctx[b]):
            t = int(c["table"][b, p // page])
            if 0 <= t < used.shape[0]:
                used[t, p % page] = True
    raw = (torch.uint8, 0x7f) if fmt == "e4m3" else (torch.int16, 0x7fc0)
    for x in (c["kc"], c["vc"]):
        x.view(raw[0]).transpose(1, 2)[~used] = raw[1]
    if fmt == "e4m3":
        c["ks"].transpose(1, 2)[~used], c["vs"].transpose(1, 2)[~used] = math.nan, math.inf
    # drafted token 3 of sequence 3 holds NaN; only its own row and its children's see it: those are not looked at
    pos = ctx[3] + 3
    t, o = int(c["table"][3, pos // page]), pos % page
    c["bits"][13 + 4:13 + 20, 0] &= ~(1 << 3)
    clean = {x: None if y is None else y.clone() for x, y in c.items()}
    for x in (c["kc"], c["vc"]):
        x.view(raw[0])[t, :, o] = raw[1]
    c["vc"].view(raw[0])[t, :, o, ::2] = 0x7f80 if fmt == "bf16" else 0xff
    out, lse = _run_tree(ext, c, dev)
    torch.cuda.synchronize()
    N, HQ = out.shape[0], 6
    dirty = 13 + 3
    assert bool(torch.isnan(out[dirty].float()).any())
    clean_out, clean_lse = _run_tree(ext, clean, dev)
    keep = [i for i in range(N) if i != dirty]
    _check_tree(C, clean, clean_out, clean_lse, D ** -0.5)
    out, lse = out.clone(), lse.clone()
    out[dirty], lse[dirty] = clean_out[dirty], clean_lse[dirty]
    _check_tree(C, clean, out, lse, D ** -0.5)
    assert bool((out[2] == 0).all()) and bool((out[6] == 0).all()) and bool((out[-3:] == 0).all())
    assert bool((lse[2] == -math.inf).all()) and bool((lse[-3:] == -math.inf).all()) and len(keep) == N - 1


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("n,G", [(5, 2), (14, 4), (40, 5)])
def test_tree_attn_unseen_places_change_nothing(ext, dev, n, G, fmt):
    """The same bits whatever lies in places that no row sees: free pages, places behind the sequences' ends, pages that the
    table names wrongly, drafted tokens that no row has a bit for. Row blocks of 16, 64 and 128."""
    _say(f"case unseen {n} {G} {fmt}")
    page, D = 32, 256
    c = _tree_case([n, n], [300, 45], 2, G, D, page, fmt, dev, seed=n, ext=ext)
    c["bits"][:, 0] &= ~(1 << 2)               # drafted token 2: nobody's, not even its own
    lost = int(c["table"][0, 3])
    c["table"][0, 3] = -1
    seen = torch.zeros(c["kc"].shape[0], page, dtype=torch.bool)
    for b, ctx in enumerate((300, 45)):
        for p in range(ctx + n):
            if int(c["table"][b, p // page]) >= 0 and p != ctx + 2:
                seen[int(c["table"][b, p // page]), p % page] = True
    assert not bool(seen[lost].any())
    want = _run_tree(ext, c, dev)
    raw, bad = (torch.uint8, 0x7f) if fmt == "e4m3" else (torch.int16, 0x7fc0)
    for x in (c["kc"], c["vc"]):
        x.view(raw).transpose(1, 2)[~seen] = bad
    # the values of a drafted token that rows do see elsewhere stay numbers: those that are not go one by one, in another order
    for b, ctx in enumerate((300, 45)):
        t, o = int(c["table"][b, (ctx + 2) // page]), (ctx + 2) % page
        c["vc"][t, :, o] = torch.full((), 7.0).to(c["vc"].dtype)
    if fmt == "e4m3":
        c["ks"].transpose(1, 2)[~seen], c["vs"].transpose(1, 2)[~seen] = math.nan, math.inf
    got = _run_tree(ext, c, dev)
    assert bool(torch.isfinite(want[0].float()).all())
    assert torch.equal(got[0].view(torch.int16), want[0].view(torch.int16)) and torch.equal(got[1], want[1])


def test_tree_attn_table_ends_early(ext, C, dev):
    """Positions past max_pages * page are not seen, drafted ones among them."""
    c = _tree_case([6], [60], 2, 3, 128, 16, "bf16", dev, seed=5, ext=ext)
    c["table"] = c["table"][:, :4].contiguous()      # 64 of 66 positions
    out, lse = _run_tree(ext, c, dev)
    _check_tree(C, c, out, lse, 128 ** -0.5)
    none = dict(c, table=c["table"][:, :0].contiguous())
    out, lse = _run_tree(ext, none, dev)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


def test_tree_attn_odd_pointers(ext, dev):
    """Pointers outside the rows, falling ones and negative lengths stay within the tensors; rows of no sequence give
    zeros."""
    c = _tree_case([4, 4], [20, 30], 1, 2, 128, 16, "bf16", dev, seed=6, ext=ext)
    for ptr, ctx in (([-7, 4, 900], [20, 30]), ([0, 6, 2], [20, 30]), ([3, 5, 7], [-4, 1 << 30]),
                     ([0, 4, 8], [(1 << 31) - 1, -(1 << 31)])):
        c["q_ptr"], c["ctx"] = torch.tensor(ptr, dtype=torch.int32), torch.tensor(ctx, dtype=torch.int32)
        out, lse = _run_tree(ext, c, dev)
        torch.cuda.synchronize()
        assert bool(torch.isfinite(out.float()).all()) and not bool(torch.isnan(lse).any())
    c["q_ptr"], c["ctx"] = torch.tensor([3, 5, 7], dtype=torch.int32), torch.tensor([20, 30], dtype=torch.int32)
    out, lse = _run_tree(ext, c, dev)
    assert bool((out[[0, 1, 2, 7]] == 0).all()) and bool((lse[[0, 1, 2, 7]] == -math.inf).all())
    assert bool((out[3:7] != 0).any(1).all())


SHARES = [
    # drafted, cached, HKV, G, D, page: how row blocks and positions are shared out
    ([1 + i % 3 for i in range(70)], [(i * 37) % 200 for i in range(69)] + [3001], 16, 2, 128, 64),   # more blocks than a round
    ([8 + i % 13 for i in range(20)], [(i * 53) % 700 for i in range(20)], 16, 4, 128, 64),           # 64 rows, one round
    ([10] * 66, [100] * 65 + [1500], 16, 4, 128, 64),                                                 # 64 rows, more blocks
    ([0] * 30 + [12, 3] + [0] * 60 + [20, 9], [5] * 30 + [900, 70] + [40] * 60 + [0, 333], 4, 6, 128, 32),  # empty ones
    ([40, 70, 33], [650, 31, 1200], 2, 4, 256, 64),                                                   # 128 rows
    ([1] * 64, [640] * 64, 4, 6, 256, 64),                                                            # equal, decoding
]


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("case", range(len(SHARES)))
def test_tree_attn_shares(ext, C, dev, case, fmt):
    n, ctx, HKV, G, D, page = SHARES[case]
    _say(f"case shares {case} {fmt}")
    c = _tree_case(n, ctx, HKV, G, D, page, fmt, dev, seed=100 + case, ext=ext)
    out, lse = _run_tree(ext, c, dev)
    _check_tree(C, c, out, lse, D ** -0.5)


def test_tree_attn_more_parts_than_lanes(ext, dev):
    """A context of more parts than a wave has lanes; with no scale, every weight is the same: the values' mean."""
    ctx, D = 20011, 128
    c = _tree_case([1], [ctx], 1, 2, D, 64, "bf16", dev, seed=8, chain=True, ext=ext)
    out, lse = _run_tree(ext, c, dev, 0.0)
    t = torch.arange(ctx + 1)
    v = c["vc"][c["table"][0].long()[t // 64], 0, t % 64].double()
    # fp32 sums of 20012 values in some order, then a division and a rounding to bf16 (half a step is 2^-8)
    bound = (v.abs().mean(0) * (ctx + 3) * 2.0 ** -24 + v.mean(0).abs() * 2.0 ** -8) * 1.01
    for h in range(2):
        assert bool(((out[0, h * D:(h + 1) * D].cpu().double() - v.mean(0)).abs() <= bound).all())
    assert abs(lse[0, 0].item() - math.log(ctx + 1)) <= math.log(ctx + 1) * 2.0 ** -21


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("n,G", [(5, 2), (14, 4), (40, 5)])
def test_tree_attn_values_not_finite(ext, dev, n, G, fmt):
    """With no scale every weight is one: an infinity (a NaN in e4m3) in the context reaches every row, one in a drafted
    token the rows that see it; in their own dim only, and nothing else changes. Row blocks of 16, 64 and 128."""
    _say(f"case values {n} {G} {fmt}")
    ctx, page, D = 700, 64, 256
    c = _tree_case([n], [ctx], 2, G, D, page, fmt, dev, seed=n, ext=ext)
    clean, clean_lse = _run_tree(ext, c, dev, 0.0)
    see = [bool(int(c["bits"][i, 0]) >> 2 & 1) for i in range(n)]  # who sees drafted token 2
    assert any(see) and not all(see)
    raw, hi, lo = (torch.uint8, 0x7f, 0xff) if fmt == "e4m3" else (torch.int16, 0x7f80, 0xff80 - 65536)
    for pos, d, x in ((5, 3, hi), (ctx + 2, 7, lo)):
        c["vc"].view(raw)[int(c["table"][0, pos // page]), :, pos % page, d] = x
    out, lse = _run_tree(ext, c, dev, 0.0)
    got, want = out.view(n, 2 * G, D).float().cpu(), clean.view(n, 2 * G, D).float().cpu()
    bad = torch.zeros(n, 2 * G, D, dtype=torch.bool)
    bad[..., 3] = True
    bad[torch.tensor(see), :, 7] = True
    if fmt == "bf16":
        assert bool((got[..., 3] == math.inf).all()) and bool((got[torch.tensor(see), :, 7] == -math.inf).all())
    else:
        assert bool(torch.isnan(got[bad]).all())
    assert torch.equal(got[~bad], want[~bad]) and torch.equal(lse, clean_lse)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("n,G", [(5, 2), (14, 4), (40, 5)])
def test_tree_attn_values_not_finite_of_no_weight(ext, dev, n, G, fmt):
    """A value that is not finite reaches every row that sees it, also where its weight is too small for fp32: scores of
    -256 beside scores around zero. Of a drafted token and of the context's last one; row blocks of 16, 64 and 128."""
    _say(f"case no weight {n} {G} {fmt}")
    ctx, page, D = 700, 64, 256
    c = _tree_case([n], [ctx], 2, G, D, page, fmt, dev, seed=n, ext=ext)
    c["q"].fill_(1)
    at = [(int(c["table"][0, pos // page]), pos % page) for pos in (ctx + 2, ctx - 1)]
    for t, o in at:
        c["kc"].view(torch.uint8 if fmt == "e4m3" else torch.int16)[t, :, o] = 0xd8 if fmt == "e4m3" else 0xc180 - 65536  # -16
        if fmt == "e4m3":
            c["ks"][t, :, o] = 1.0
    clean, clean_lse = _run_tree(ext, c, dev)
    see = torch.tensor([bool(int(c["bits"][i, 0]) >> 2 & 1) for i in range(n)])
    assert bool(see.any()) and not bool(see.all())
    raw, inf = (torch.uint8, 0x7f) if fmt == "e4m3" else (torch.int16, 0x7f80)
    for (t, o), d in zip(at, (7, 3)):
        c["vc"].view(raw)[t, :, o, d] = inf
    out, lse = _run_tree(ext, c, dev)
    got, want = out.view(n, 2 * G, D).float().cpu(), clean.view(n, 2 * G, D).float().cpu()
    bad = torch.zeros(n, 2 * G, D, dtype=torch.bool)
    bad[see, :, 7] = True
    bad[..., 3] = True
    assert bool(torch.isfinite(want).all()) and not bool(torch.isfinite(got[bad]).any())
    assert torch.equal(got[~bad], want[~bad]) and torch.equal(lse, clean_lse)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("n,G", [(5, 2), (14, 4), (40, 5)])
def test_tree_attn_keys_not_finite(ext, dev, n, G, fmt):
    """A NaN in a drafted token's key makes the rows that see it NaN, lse included, and changes no bit of the others."""
    _say(f"case keys {n} {G} {fmt}")
    ctx, page, D = 700, 64, 128
    c = _tree_case([n, 3], [ctx, 40], 2, G, D, page, fmt, dev, seed=n, ext=ext)
    want, want_lse = _run_tree(ext, c, dev)
    see = torch.tensor([bool(int(c["bits"][i, 0]) >> 2 & 1) for i in range(n)] + [False] * 3)
    assert bool(see.any()) and not bool(see[:n].all())
    raw, bad = (torch.uint8, 0x7f) if fmt == "e4m3" else (torch.int16, 0x7fc0)
    c["kc"].view(raw)[int(c["table"][0, (ctx + 2) // page]), :, (ctx + 2) % page, 9] = bad
    out, lse = _run_tree(ext, c, dev)
    see = see.to(dev)
    assert bool(torch.isnan(out[see].float()).all()) and bool(torch.isnan(lse[see]).all())
    assert torch.equal(out[~see], want[~see]) and torch.equal(lse[~see], want_lse[~see])


@pytest.mark.parametrize("n,D", [(1, 256), (6, 128), (30, 256)])
def test_tree_attn_graph_of_growing_contexts(ext, dev, n, D):
    """One captured call, replayed while the contexts on the device grow and shrink: lengths are looked at on the device,
    so every replay is the eager call's result for the lengths of the moment."""
    c = _tree_case([n, n], [900, 1500], 2, 4, D, 64, "bf16", dev, seed=n, ext=ext)
    d = {x: None if t is None else t.to(dev) for x, t in c.items()}
    call = lambda: ext.tree_attn(d["q"], d["kc"], d["vc"], d["table"], d["ctx"], d["q_ptr"], d["bits"], want_lse=True)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = call()
    for ctx in ([900, 1500], [0, 31], [17, 1500], [899, 2], [900, 1499]):
        d["ctx"].copy_(torch.tensor(ctx, dtype=torch.int32))
        want, want_lse = call()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, want_lse)


def test_tree_attn_empty(ext, dev):
    c = _tree_case([2], [20], 1, 2, 128, 16, "bf16", dev, seed=7, ext=ext)
    c["q"], c["bits"] = c["q"][:, :0].contiguous(), c["bits"][:0].contiguous()
    c["q_ptr"].zero_()
    out, lse = _run_tree(ext, c, dev)
    assert tuple(out.shape) == (0, 256) and tuple(lse.shape) == (0, 2)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("page", [16, 112, 240, 1008, 1024])
def test_tree_attn_pages(ext, C, dev, page, fmt):
    """The smallest and the largest page, and some that are no power of two: where a position lies is a division."""
    _say(f"case page {page} {fmt}")
    c = _tree_case([3, 1, 21], [0, 1030, 257], 1, 4, 128, page, fmt, dev, seed=page, ext=ext)
    out, lse = _run_tree(ext, c, dev)
    _check_tree(C, c, out, lse, 128 ** -0.5)


def test_cores_without_sequences(ext, dev):
    """Rows and no sequence at all: zeros (lse -inf), and no states."""
    c = _tree_case([4], [20], 2, 3, 256, 16, "bf16", dev, seed=9, ext=ext)
    for pages in (2, 400):
        none = dict(c, ctx=c["ctx"][:0], q_ptr=c["q_ptr"][:1], table=torch.zeros(0, pages, dtype=torch.int32))
        out, lse = _run_tree(ext, none, dev)
        assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    for delta in (True, False):
        o, last = ext.linattn_prompt(*_put(dev, *_lin_case(200, 1, 3, delta, seed=9), torch.zeros(1, dtype=torch.int32)))
        assert bool((o == 0).all()) and tuple(last.shape) == (0, 3, 128, 128)


def test_tree_attn_long(ext, C, dev):
    """A long context, checked on a few rows: every split of it and their join."""
    for fmt, n, ctx in (("e4m3", 1, 20011), ("bf16", 13, 9001)):
        _say(f"case long {fmt}")
        c = _tree_case([n], [ctx], 1, 6, 256, 64, fmt, dev, seed=ctx, ext=ext)
        out, lse = _run_tree(ext, c, dev)
        one = dict(c, q=c["q"][:, n - 1:].contiguous(), bits=c["bits"][n - 1:].contiguous())
        # row n - 1 alone: its drafted predecessors stand at their places behind the context
        K, V = C.cache_values(c["kc"], c["ks"]), C.cache_values(c["vc"], c["vs"])
        pos = [p for p in range(ctx + n) if p < ctx or (int(c["bits"][n - 1, 0]) >> (p - ctx)) & 1]
        t = torch.tensor(pos)
        page, off = c["table"][0].long()[t // 64], t % 64
        for h in range(6):
            k, v, x = K[page, 0, off], V[page, 0, off], one["q"][h, 0].double()
            s = (k @ x) / 16
            w = torch.softmax(s, 0)
            es = ((k.abs() @ x.abs()) / 16 * 264 * C.F + (s.abs() + s.abs().max() + 8) * 4 * C.F).max().item()
            bound = (w @ v.abs()) * (C.U + 2 * es + 2 * len(pos) * C.F) * 1.01 + C.U * (w @ v).abs() * 1.01
            got = out[n - 1, h * 256:(h + 1) * 256].cpu().double()
            assert bool(((got - w @ v).abs() <= bound).all())
            assert abs(lse[n - 1, h].item() - torch.logsumexp(s, 0).item()) <= es + len(pos) * C.F + 1e-5


# ----------------------------------------------------------------------------------------------------- linear attention
def _lin_case(R, HK, G, delta, seed, sharp=False):
    """Operands as the prep gives them. sharp: decays from none at all to a cleared state, strengths of 0 and 1, keys that
    repeat."""
    g = torch.Generator().manual_seed(seed)
    HV = HK * G
    qk = torch.nn.functional.silu(torch.randn(2, R, HK, 128, generator=g) + 0.3)
    if sharp and R > 3:
        qk[1, 1::3] = qk[1, :1]
    qk = (qk / (qk.square().sum(-1, keepdim=True) + 1e-6).sqrt()).bfloat16().reshape(2, R, HK * 128)
    v = torch.nn.functional.silu(torch.randn(R, HV * 128, generator=g)).bfloat16()
    gate = -torch.rand(R, HV, generator=g) * torch.exp(3 * torch.randn(HV, generator=g) - 2)
    beta = torch.sigmoid(2 * torch.randn(R, HV, generator=g)).bfloat16()
    if sharp:
        pick = torch.rand(R, HV, generator=g)
        gate = torch.where(pick < 0.3, torch.zeros(()), gate)
        gate = torch.where(pick > 0.97, torch.full((), -math.inf), torch.where(pick > 0.94, torch.full((), -150.0), gate))
        beta = torch.where(torch.rand(R, HV, generator=g) < 0.2, torch.ones(()), beta.float()).bfloat16()
        beta = torch.where(torch.rand(R, HV, generator=g) < 0.2, torch.zeros(()), beta.float()).bfloat16()
    return qk[0].contiguous(), qk[1].contiguous(), v, gate, beta if delta else None


def _put(dev, *ts):
    return [None if t is None else t.to(dev) for t in ts]


def _check_lin(C, args, lengths, state, got_o, got_s, scale):
    o, st, bo, bs = C.linattn(*args, lengths, state, scale)
    R = sum(lengths)
    err = (got_o[:R].cpu().double().reshape(o[:R].shape) - o[:R]).abs()
    worst = (err / bo[:R].clamp_min(1e-300)).max().item() if R else 0.0
    es = (got_s.cpu().double() - st).norm(dim=(2, 3))
    worse = (es / bs.clamp_min(1e-300)).max().item() if bool((bs > 0).any()) else 0.0
    _say(f"  out {worst:.3f}, state {worse:.3f} of the bounds; state off by {(es.norm() / st.norm().clamp_min(1e-30)).item():.2e}")
    assert bool((err <= bo[:R]).all()), f"out: {worst:.3f} of the bound"
    assert bool((es <= bs).all()), f"state: {worse:.3f} of the bound"


PROMPTS = [
    # lengths, HK, G
    ([1], 1, 1), ([2], 1, 3), ([63], 2, 1), ([64], 1, 2), ([65], 2, 3), ([0, 5, 0], 1, 1), ([130, 1, 64, 17], 1, 3),
    ([288], 2, 3), ([16] * 9, 1, 2), ([31, 33, 32, 127, 128, 129], 1, 1),
]


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("case", range(len(PROMPTS)))
def test_linattn_prompt(ext, C, dev, case, delta):
    lengths, HK, G = PROMPTS[case]
    for sharp in (False, True):
        for start in (False, True):
            _say(f"case prompt {case} delta={delta} sharp={sharp} start={start}")
            R, S, HV = sum(lengths), len(lengths), HK * G
            args = _lin_case(R, HK, G, delta, seed=case, sharp=sharp)
            ptr = torch.tensor([0] + list(torch.tensor(lengths).cumsum(0)), dtype=torch.int32)
            pool = src = state = None
            if start:
                pool = torch.randn(S + 2, HV, 128, 128, generator=torch.Generator().manual_seed(case)) * 0.1
                src = torch.tensor([(3 * s) % (S + 2) if s % 3 else -1 for s in range(S)], dtype=torch.int32)
                state = torch.where((src >= 0)[:, None, None, None], pool[src.clamp_min(0).long()], torch.zeros(()))
            o, last = ext.linattn_prompt(*_put(dev, *args, ptr, pool, src))
            _check_lin(C, args, lengths, state, o, last, 128 ** -0.5)


def test_linattn_prompt_rows_of_no_sequence(ext, C, dev):
    """Rows before the first and behind the last sequence give zeros, whatever they hold; pointers out of range stay
    within the rows; a source outside the states gives NaN."""
    args = _lin_case(100, 1, 2, True, seed=1)
    for t in args[:3]:
        t[:7], t[90:] = math.nan, math.inf
    args[3][:7], args[3][90:] = math.nan, math.nan
    ptr = torch.tensor([7, 40, 90], dtype=torch.int32)
    o, last = ext.linattn_prompt(*_put(dev, *args, ptr))
    assert bool((o[:7] == 0).all()) and bool((o[90:] == 0).all())
    inner = [t[7:90].contiguous() for t in args]
    _check_lin(C, inner, [33, 50], None, o[7:90], last, 128 ** -0.5)
    args = _lin_case(20, 1, 2, True, seed=2)
    for odd in ([-9, 10, 400], [0, 15, 3], [30, 40, 50]):
        o, last = ext.linattn_prompt(*_put(dev, *args, torch.tensor(odd, dtype=torch.int32)))
        torch.cuda.synchronize()
        assert bool(torch.isfinite(o.float()).all()) and bool(torch.isfinite(last).all())
    pool = torch.ones(2, 2, 128, 128)
    o, last = ext.linattn_prompt(*_put(dev, *args, torch.tensor([0, 10, 20], dtype=torch.int32), pool,
                                       torch.tensor([2, 0], dtype=torch.int32)))
    assert bool(torch.isnan(last[0]).all()) and bool(torch.isfinite(last[1]).all())
    assert bool(torch.isnan(o[:10].float()).all()) and bool(torch.isfinite(o[10:].float()).all())


def test_linattn_nan_stays_in_its_sequence_and_head(ext, dev):
    args = _lin_case(140, 1, 3, True, seed=3)
    clean = ext.linattn_prompt(*_put(dev, *args, torch.tensor([0, 70, 140], dtype=torch.int32)))
    bad = [t.clone() for t in args]
    bad[2][20, 128:256] = math.nan          # value head 1 of sequence 0
    o, last = ext.linattn_prompt(*_put(dev, *bad, torch.tensor([0, 70, 140], dtype=torch.int32)))
    o, c = o.reshape(140, 3, 128).float(), clean[0].reshape(140, 3, 128).float()
    assert torch.equal(o[:, [0, 2]], c[:, [0, 2]]) and torch.equal(o[70:], c[70:])
    assert bool(torch.isnan(o[20:70, 1]).all()) and bool(torch.isnan(last[0, 1]).all())
    assert torch.equal(last[1], clean[1][1]) and torch.equal(last[0, [0, 2]], clean[1][0, [0, 2]])
    bad = [t.clone() for t in args]
    bad[3][80, 2] = math.nan                # a decay
    o, last = ext.linattn_prompt(*_put(dev, *bad, torch.tensor([0, 70, 140], dtype=torch.int32)))
    assert bool(torch.isnan(last[1, 2]).all()) and torch.equal(last[0], clean[1][0])
    assert bool(torch.isnan(o.reshape(140, 3, 128)[80:, 2].float()).all())


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("R,HK,G", [(1, 1, 1), (1, 16, 3), (5, 2, 3), (33, 1, 2)])
def test_linattn_step(ext, C, dev, R, HK, G, delta):
    _say(f"case step R={R} HK={HK} G={G} delta={delta}")
    HV = HK * G
    args = _lin_case(R, HK, G, delta, seed=R, sharp=R > 4)
    g = torch.Generator().manual_seed(R)
    pool = torch.randn(R + 3, HV, 128, 128, generator=g) * 0.1
    slot = torch.randperm(R + 3, generator=g)[:R].int()
    if R > 4:
        slot[1], slot[3], slot[4] = -1, R + 3, slot[0]      # idle, not there, named twice
    d = _put(dev, *args, pool, slot)
    o = ext.linattn_step(*d)
    torch.cuda.synchronize()
    runs = [r for r in range(R) if R <= 4 or r not in (1, 3, 4)]
    rows = [None if t is None else t[runs].contiguous() for t in args]
    at = slot[runs].long()
    got = d[5].cpu()
    _check_lin(C, rows, [1] * len(runs), pool[at], o[runs], got[at], 128 ** -0.5)
    rest = torch.ones(R + 3, dtype=torch.bool)
    rest[at] = False
    assert torch.equal(got[rest], pool[rest])
    if R > 4:
        assert bool((o[1] == 0).all()) and bool(torch.isnan(o[3].float()).all()) and bool(torch.isnan(o[4].float()).all())


@pytest.mark.parametrize("delta", [True, False])
def test_linattn_step_of_slots_named_again(ext, C, dev, delta):
    """The first row that names a slot has it; every later one is NaN and leaves the states alone. Rows apart by less and
    by more than a workgroup's 256 threads, a slot named three times, idle rows between."""
    R = 600
    args = _lin_case(R, 1, 1, delta, seed=81)
    g = torch.Generator().manual_seed(81)
    pool = torch.randn(R + 40, 1, 128, 128, generator=g) * 0.1
    slot = torch.randperm(R + 40, generator=g)[:R].int()
    again = {10: 3, 70: 3, 200: 100, 255: 0, 256: 1, 257: 2, 300: 5, 511: 255 + 45, 513: 254, 560: 520, 598: 256 + 7, 599: 597}
    for r, of in again.items():
        slot[r] = slot[of]                     # row 511 names what row 300 took from row 5
    idle = [4, 63, 64, 258, 512]
    slot[idle[:3]], slot[idle[3:]] = -1, -(1 << 31)
    assert int(slot[511]) == int(slot[5])
    d = _put(dev, *args, pool, slot)
    o = ext.linattn_step(*d).cpu()
    got = d[5].cpu()
    runs = [r for r in range(R) if r not in again and r not in idle]
    assert len({int(slot[r]) for r in runs}) == len(runs)
    at = slot[runs].long()
    _check_lin(C, [None if t is None else t[runs].contiguous() for t in args], [1] * len(runs), pool[at], o[runs], got[at],
               128 ** -0.5)
    rest = torch.ones(R + 40, dtype=torch.bool)
    rest[at] = False
    assert torch.equal(got[rest], pool[rest])
    assert bool(torch.isnan(o[list(again)].float()).all()) and bool((o[idle] == 0).all())


def test_linattn_steps_go_on_from_a_prompt(ext, C, dev):
    """A prompt, then single tokens on its states, against the oracle's whole sequences."""
    lengths, more, HK, G = [70, 3, 129], 5, 1, 3
    S, HV = 3, 3
    whole = _lin_case(sum(lengths) + S * more, HK, G, True, seed=9)
    bounds = [0]
    for x in lengths:
        bounds.append(bounds[-1] + x + more)
    head = torch.cat([torch.arange(bounds[s], bounds[s] + lengths[s]) for s in range(S)])
    ptr = torch.tensor([0] + list(torch.tensor(lengths).cumsum(0)), dtype=torch.int32)
    o1, st = ext.linattn_prompt(*_put(dev, *[t[head].contiguous() for t in whole], ptr))
    outs = torch.zeros(bounds[-1], HV * 128, dtype=torch.bfloat16)
    outs[head] = o1.cpu()
    slot = torch.arange(S, dtype=torch.int32, device=dev)
    for j in range(more):
        rows = torch.tensor([bounds[s] + lengths[s] + j for s in range(S)])
        outs[rows] = ext.linattn_step(*_put(dev, *[t[rows].contiguous() for t in whole]), st, slot).cpu()
    _check_lin(C, whole, [x + more for x in lengths], None, outs, st, 128 ** -0.5)


def test_linattn_long_and_many(ext, C, dev):
    """A long sequence in one head, and many short ones: the chunks' order and the sequences' bounds."""
    args = list(_lin_case(1500, 1, 1, True, seed=21))
    args[3] = -0.02 * torch.rand(1500, 1, generator=torch.Generator().manual_seed(21))    # a memory of about 100 tokens
    o, last = ext.linattn_prompt(*_put(dev, *args, torch.tensor([0, 1500], dtype=torch.int32)))
    _check_lin(C, args, [1500], None, o, last, 128 ** -0.5)
    lengths = [(i * 37) % 71 for i in range(40)]
    args = _lin_case(sum(lengths), 1, 1, True, seed=22)
    ptr = torch.tensor([0] + list(torch.tensor(lengths).cumsum(0)), dtype=torch.int32)
    o, last = ext.linattn_prompt(*_put(dev, *args, ptr))
    _check_lin(C, args, lengths, None, o, last, 128 ** -0.5)


def test_falling_pointers_do_not_multiply_rows(ext, C, dev):
    """Pointers that fall give sequences that begin where those before them ended: no row twice, no more chunks or row
    blocks than there are rows for."""
    R = 130
    args = _lin_case(R, 1, 2, True, seed=31)
    up = [0, R, 0, R, 5, R, 0, R, 129, R]
    o, last = ext.linattn_prompt(*_put(dev, *args, torch.tensor(up, dtype=torch.int32)))
    _check_lin(C, args, [R] + [0] * 8, None, o, last, 128 ** -0.5)
    up = [0, 70, 10, 90, 20, 130]
    o, last = ext.linattn_prompt(*_put(dev, *args, torch.tensor(up, dtype=torch.int32)))
    _check_lin(C, args, [70, 0, 20, 0, 40], None, o, last, 128 ** -0.5)
    c = _tree_case([40], [30], 1, 2, 128, 16, "bf16", dev, seed=31, ext=ext)
    c["table"] = c["table"].repeat(4, 1).contiguous()
    c["ctx"] = c["ctx"].repeat(4).contiguous()
    want = dict(c, q_ptr=torch.tensor([0, 40, 40, 40, 40], dtype=torch.int32))
    c["q_ptr"] = torch.tensor([0, 40, 0, 40, 0], dtype=torch.int32)
    out, lse = _run_tree(ext, c, dev)
    _check_tree(C, want, out, lse, 128 ** -0.5)


def test_linattn_prompt_without_rows(ext, dev):
    """Sequences without rows hand their states on."""
    args = _put(dev, *_lin_case(0, 1, 2, True, seed=1))
    pool = torch.randn(3, 2, 128, 128, device=dev)
    o, last = ext.linattn_prompt(*args, torch.zeros(3, dtype=torch.int32, device=dev), pool,
                                 torch.tensor([2, -1], dtype=torch.int32, device=dev))
    assert tuple(o.shape) == (0, 256) and torch.equal(last[0], pool[2]) and bool((last[1] == 0).all())


def test_linattn_prompt_of_an_empty_pool(ext, C, dev):
    """A pool of no states has none to start from: sequences that name one are NaN, as with every source outside the
    states, and the others start from zeros."""
    args = _lin_case(30, 1, 2, True, seed=4)
    ptr, src = torch.tensor([0, 10, 30], dtype=torch.int32), torch.tensor([-1, 0], dtype=torch.int32)
    o, last = ext.linattn_prompt(*_put(dev, *args, ptr, torch.zeros(0, 2, 128, 128), src))
    assert bool(torch.isnan(last[1]).all()) and bool(torch.isnan(o[10:].float()).all())
    _check_lin(C, [t[:10].contiguous() for t in args], [10], None, o[:10], last[:1], 128 ** -0.5)


# ------------------------------------------------------------- many heads: a workgroup of eight waves a sequence and head
_SHORT = [0, 1, 64, 3, 65, 17, 130, 63, 2, 33]
MANY = [
    # lengths, HK, G: sequences times value heads on both sides of 96, where the form for many heads begins
    (_SHORT * 9 + _SHORT[4:], 1, 1),                 # 96: the last of the form for few
    (_SHORT * 9 + _SHORT[3:], 1, 1),                 # 97, a head each: no multiple of the eight XCDs
    ((_SHORT * 4)[:33], 1, 3),                       # 99
    ([65, 0, 200, 64, 1, 63, 129], 5, 3),            # 105, of 35 key heads
    ([70, 0, 65], 16, 3),                            # 144: the model's heads
    ([0] * 100 + [5], 1, 2),                         # all but one empty
]


def _many_case(case, delta, lead=5, tail=9):
    """Rows of no sequence before and behind the sequences, NaN in them; every third sequence from zeros, one from a state
    that is not there, the others from a pool's."""
    lengths, HK, G = MANY[case]
    R, S, HV = sum(lengths), len(lengths), HK * G
    args = _lin_case(lead + R + tail, HK, G, delta, seed=50 + case, sharp=case % 2 == 1)
    for t in args:
        if t is not None:
            t[:lead], t[lead + R:] = math.nan, math.nan
    ptr = torch.tensor([lead] + list(lead + torch.tensor(lengths).cumsum(0)), dtype=torch.int32)
    pool = torch.randn(S + 2, HV, 128, 128, generator=torch.Generator().manual_seed(case)) * 0.1
    src = torch.tensor([(3 * s) % (S + 2) if s % 3 else -1 for s in range(S)], dtype=torch.int32)
    src[S // 2] = S + 2
    return args, ptr, pool, src


def _check_many(C, args, ptr, pool, src, o, last):
    """Against the oracle; sequences from states that are not there are NaN, and the rows of no sequence zeros."""
    lead, S = int(ptr[0]), ptr.numel() - 1
    lengths = (ptr[1:] - ptr[:-1]).tolist()
    end = lead + sum(lengths)
    o, last = o.cpu(), last.cpu()
    assert bool((o[:lead] == 0).all()) and bool((o[end:] == 0).all())
    state = None
    if pool is not None:
        state = torch.where((src >= 0)[:, None, None, None], pool[src.clamp(0, pool.shape[0] - 1).long()], torch.zeros(()))
        for s in range(S):
            if int(src[s]) >= pool.shape[0]:
                at = slice(int(ptr[s]), int(ptr[s + 1]))
                assert bool(torch.isnan(last[s]).all()) and bool(torch.isnan(o[at].float()).all())
                # for the comparison below, as if it had started from zeros
                state[s] = last[s] = 0
                if lengths[s] == 0:
                    continue
                sub = [None if t is None else t[at].contiguous() for t in args]
                ro, rs, _, _ = C.linattn(*sub, [lengths[s]], None, 128 ** -0.5)
                o[at], last[s] = ro.reshape(ro.shape[0], -1).bfloat16(), rs[0].float()
    inner = [None if t is None else t[lead:end].contiguous() for t in args]
    _check_lin(C, inner, lengths, state, o[lead:end], last, 128 ** -0.5)


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("case", range(len(MANY)))
def test_linattn_prompt_many(ext, C, dev, case, delta):
    _say(f"case many {case} delta={delta}")
    args, ptr, pool, src = _many_case(case, delta)
    o, last = ext.linattn_prompt(*_put(dev, *args, ptr, pool, src))
    _check_many(C, args, ptr, pool, src, o, last)
    o, last = ext.linattn_prompt(*_put(dev, *args, ptr))
    _check_many(C, args, ptr, None, None, o, last)


@pytest.mark.parametrize("delta", [True, False])
def test_linattn_prompt_many_falling_pointers(ext, C, dev, delta):
    """Pointers in no order, some outside the rows: sequences begin where those before them ended."""
    R, S = 400, 120
    g = torch.Generator().manual_seed(61)
    args = _lin_case(R, 1, 2, delta, seed=61)
    raw = (torch.arange(S + 1) * 4 + torch.randint(-60, 60, (S + 1,), generator=g)).int()
    raw[0], raw[50], raw[-1] = 3, 1 << 30, -7
    raw[51:] = torch.randint(-500, 500, (S - 50,), generator=g).int()
    raw[49] = 250
    at = raw.clamp(0, R).cummax(0).values
    o, last = ext.linattn_prompt(*_put(dev, *args, raw))
    _check_many(C, args, at, None, None, o, last)


@pytest.mark.parametrize("delta", [True, False])
def test_linattn_prompt_many_not_finite(ext, C, dev, delta):
    """A value that is not finite in the middle chunk of one of many sequences: what it reaches by the formula is not
    finite, and everything else is the oracle's, in the chunks behind it, too."""
    lengths, HK, G = [30] * 16 + [200] + [30] * 17, 1, 3
    R, HV = sum(lengths), 3
    args = _lin_case(R, HK, G, delta, seed=71)
    ptr = torch.tensor([0] + list(torch.tensor(lengths).cumsum(0)), dtype=torch.int32)
    first, at = int(ptr[16]), int(ptr[16]) + 100
    o, st, bo, bs = C.linattn(*args, lengths, None, 128 ** -0.5)
    for which, value in (("q", math.inf), ("k", math.nan), ("v", math.nan), ("v", -math.inf), ("g", math.nan),
                         ("g", math.inf), ("beta", math.inf)):
        if which == "beta" and not delta:
            continue
        _say(f"case many not finite {which} {value} delta={delta}")
        bad = [None if t is None else t.clone() for t in args]
        hit = torch.zeros(R, HV, 128, dtype=torch.bool)        # outputs that are not finite
        lost = torch.zeros(HV, 128, dtype=torch.bool)          # value dims of the sequence's state
        if which == "q":
            bad[0][at, 5] = value
            hit[at] = True
        elif which == "k":
            bad[1][at, 5] = value
            hit[at:first + 200], lost[:] = True, True
        elif which == "v":
            bad[2][at, 128 + 37] = value
            hit[at:first + 200, 1, 37], lost[1, 37] = True, True
        else:
            bad[3 if which == "g" else 4][at, 2] = value
            hit[at:first + 200, 2], lost[2] = True, True
        out, last = (t.cpu() for t in ext.linattn_prompt(*_put(dev, *bad, ptr)))
        out = out.double().reshape(R, HV, 128)
        assert not bool(torch.isfinite(out[hit]).any()) and bool(torch.isfinite(out[~hit]).all())
        assert bool(((out - o).abs()[~hit] <= bo[~hit]).all())
        cols = last[16].transpose(1, 2)                        # [HV, value dims, key dims]
        if which == "k" and not delta:
            assert not bool(torch.isfinite(cols[..., 5]).any())
            assert bool(torch.isfinite(cols[..., :5]).all()) and bool(torch.isfinite(cols[..., 6:]).all())
        elif which == "v":
            assert not bool(torch.isfinite(cols[lost]).all(1).any())
        elif bool(lost.any()):
            assert not bool(torch.isfinite(cols[lost]).any())
        keep = torch.ones(34, HV, dtype=torch.bool)
        keep[16] = ~lost.any(1)
        err = (last.double() - st).norm(dim=(2, 3))
        assert bool((err[keep] <= bs[keep]).all())
        assert bool(torch.isfinite(cols[~lost]).all())


@pytest.mark.parametrize("delta", [True, False])
def test_linattn_prompt_many_in_a_graph(ext, dev, delta):
    """A captured call, replayed over other inputs and pointers, with eager calls between, equals the eager call; so do
    calls on two streams at once, and the same call again."""
    args, ptr, pool, src = _many_case(2, delta)
    d = _put(dev, *args, ptr, pool, src)
    call = lambda: ext.linattn_prompt(*d)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, last = call()
    other = _put(dev, *_many_case(2, delta)[0])
    for x in other[:3]:
        x.mul_(0.5)
    for i, lengths in enumerate(([3] * 33, [0] * 32 + [400], _SHORT * 3 + [40, 64, 1])):
        d[5].copy_(torch.tensor([5] + list(5 + torch.tensor(lengths).cumsum(0)), dtype=torch.int32))
        d[2].copy_(other[2] if i % 2 == 0 else args[2])
        a, b = call(), call()
        graph.replay()
        torch.cuda.synchronize()
        for x, y, z in ((out, a[0], b[0]), (last, a[1], b[1])):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)) and torch.equal(y.view(torch.uint8), z.view(torch.uint8))
    want = call()
    torch.cuda.synchronize()
    got = []
    for s in (torch.cuda.Stream(), torch.cuda.Stream()):
        with torch.cuda.stream(s):
            got.append(call())
    torch.cuda.synchronize()
    for x in got:
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(x, want))


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("HK,G", [(2, 1), (1, 3), (4, 3), (16, 1)])
def test_linattn_prompt_keeps_its_pieces(ext, C, dev, HK, G, delta):
    """Entry by entry, sequences of up to 64 tokens from given states stay within what the pieces of the factors and fp32
    sums give (in bounds that a single piece of any factor breaks). Both forms: 18 and 27 heads, 108 and 144."""
    _say(f"case pieces HK={HK} G={G} delta={delta}")
    lengths = [1, 2, 3, 5, 8, 16, 24, 40, 64]
    args = _lin_case(sum(lengths), HK, G, delta, seed=90 + HK)
    ptr = torch.tensor([0] + list(torch.tensor(lengths).cumsum(0)), dtype=torch.int32)
    state = torch.randn(9, HK * G, 128, 128, generator=torch.Generator().manual_seed(HK))
    o, last = ext.linattn_prompt(*_put(dev, *args, ptr, state))
    want, st, bo, bs = C.linattn_chunk(*args, lengths, state, 128 ** -0.5)
    eo, es = (o.cpu().double().reshape(want.shape) - want).abs(), (last.cpu().double() - st).abs()
    _say(f"  out {(eo / bo).max().item():.3f}, state {(es / bs).max().item():.3f} of the bounds")
    assert bool((eo <= bo).all()) and bool((es <= bs).all())


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("S,HV", [(3, 2), (40, 3)])
def test_linattn_prompt_states_are_fp32(ext, C, dev, S, HV, delta):
    """States within a few steps of fp32 of 64 bits, relative to their norm, where a factor short of its third piece would
    be 13 off and more. What a chunk leaves is down to e^-0.6 after the next, so that a long sequence is off by at most
    1 / (1 - e^-0.6) = 2.2 times as much. Both forms."""
    from tests.test_cores import STATE_STEPS, slow_chunks
    _say(f"case fp32 S={S} HV={HV} delta={delta}")
    args, lengths, state = slow_chunks(S, HV, delta, 5)
    for each in ([64] * S, [64 * S] + [0] * (S - 1) if S < 10 else [64] * (S - 4) + [256, 0, 0, 0]):
        ptr = torch.tensor([0] + list(torch.tensor(each).cumsum(0)), dtype=torch.int32)
        last = ext.linattn_prompt(*_put(dev, *args, ptr, state))[1].cpu().double()
        st = C.linattn(*args, each, state, 1.0)[1]
        steps = (last - st).norm(dim=(2, 3)) / st.norm(dim=(2, 3)) / C.F
        _say(f"  {steps.max().item():.2f} steps")
        assert bool((steps <= STATE_STEPS * (1.0 if max(each) <= 64 else 2.2)).all())


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("HK,G", [(1, 3), (37, 3)])
def test_linattn_prompt_hands_its_state_on_exactly(ext, dev, HK, G, delta):
    """A long sequence is its chunks of 64 tokens in calls of their own, each from the state that the one before left, to
    the bit: what holds for one chunk holds for all. Both forms."""
    _say(f"case chunks HK={HK} G={G} delta={delta}")
    R = 64 * 5 + 9
    q, k, v, g, beta = _put(dev, *_lin_case(R, HK, G, delta, seed=95, sharp=True))
    ptr = lambda n: torch.tensor([0, n], dtype=torch.int32, device=dev)  # noqa: E731
    o, last = ext.linattn_prompt(q, k, v, g, beta, ptr(R))
    state = None
    for t in range(0, R, 64):
        r = slice(t, min(R, t + 64))
        part, state = ext.linattn_prompt(q[r], k[r], v[r], g[r], None if beta is None else beta[r], ptr(r.stop - t), state)
        assert torch.equal(part, o[r]), t
    assert torch.equal(state, last)


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("HK,G,more", [(1, 2, 0), (2, 1, 60)])
def test_linattn_prompt_decays_above_one(ext, C, dev, HK, G, more, delta):
    """A decay above 1 is no decay of these layers, but a number: chunks with one go token by token, others do not. Both
    forms."""
    _say(f"case above one HK={HK} G={G} more={more} delta={delta}")
    lengths = [200, 1, 70] + [5] * more
    args = _lin_case(sum(lengths), HK, G, delta, seed=77)
    for t, x in ((70, 0.3), (100, 1e-3), (200, 2.0), (sum(lengths) - 1, 0.05)):
        args[3][t, -1] = x
    ptr = torch.tensor([0] + list(torch.tensor(lengths).cumsum(0)), dtype=torch.int32)
    o, last = ext.linattn_prompt(*_put(dev, *args, ptr))
    _check_lin(C, args, lengths, None, o, last, 128 ** -0.5)


def test_linattn_past_32_bits(ext, dev):
    """States, rows and scratch whose offsets pass 2^32: the same bits as in a call on a few."""
    HK, HV, slots = 16, 48, 5600
    pool = torch.empty(slots, HV, 128, 128, device=dev)        # 4.4e9 values
    g = torch.Generator(device=dev).manual_seed(3)
    some = torch.randn(2, HV, 128, 128, device=dev, generator=g)
    at = torch.tensor([slots - 1, 0], dtype=torch.int32, device=dev)
    pool[at.long()] = some
    args = _put(dev, *_lin_case(140, HK, 3, True, seed=3))
    ptr = torch.tensor([0, 70, 140], dtype=torch.int32, device=dev)
    few = torch.arange(2, dtype=torch.int32, device=dev)
    a, b = ext.linattn_prompt(*args, ptr, pool, at), ext.linattn_prompt(*args, ptr, some, few)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    one = [t[:2].contiguous() for t in args]
    a, b = ext.linattn_step(*one, pool, at), ext.linattn_step(*one, some, few)
    assert torch.equal(a, b) and torch.equal(pool[at.long()], some)
    del pool
    R, tail = 360000, 300                                      # 4.4e9 bytes of v, 6.8e9 of scratch
    big = [(torch.randn(R, n, device=dev, generator=g) * 0.1).bfloat16() for n in (HK * 128, HK * 128, HV * 128)]
    big += [-torch.rand(R, HV, device=dev, generator=g), torch.rand(R, HV, device=dev, generator=g).bfloat16()]
    ends = torch.tensor([0, R - tail, R], dtype=torch.int32, device=dev)
    a = ext.linattn_prompt(*big, ends)
    b = ext.linattn_prompt(*[t[R - tail:].contiguous() for t in big], torch.tensor([0, tail], dtype=torch.int32, device=dev))
    assert torch.equal(a[0][R - tail:], b[0]) and torch.equal(a[1][1:], b[1]) and bool(torch.isfinite(a[1]).all())


def test_linattn_is_causal_in_what_is_not_finite(ext, dev):
    """NaN and infinities reach no token before theirs, in their own chunk as little as in others."""
    args = _lin_case(150, 1, 2, True, seed=33)
    ptr = torch.tensor([0, 150], dtype=torch.int32)
    clean = ext.linattn_prompt(*_put(dev, *args, ptr))[0].float()
    for t, which, value in ((20, 0, math.nan), (100, 1, math.inf), (64, 2, -math.inf), (63, 3, math.nan), (127, 4, math.nan)):
        bad = [x.clone() for x in args]
        bad[which][t] = value
        o = ext.linattn_prompt(*_put(dev, *bad, ptr))[0].float()
        err = (o[:t] - clean[:t]).abs()
        assert bool((err <= 2.0 ** -6 * clean[:t].abs().amax()).all()), which
        assert not bool(torch.isfinite(o[t]).all())


# ---------------------------------------------------------------------------------------------------- as they are used
def _layers(ext, dev, seed):
    """One decoding step's calls of a full- and a linear-attention layer, on inputs that are overwritten between calls."""
    g = torch.Generator(device=dev).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    HQ, HKV, D, n, B, page = 6, 2, 256, 4, 3, 16
    N, pages = n * B, 12
    cache = _pool(pages, HKV, page, D, "e4m3", dev)
    table = torch.arange(pages, dtype=torch.int32, device=dev).reshape(B, 4)
    ctx = torch.tensor([13, 0, 40], dtype=torch.int32, device=dev)
    q_ptr = torch.arange(0, N + 1, n, dtype=torch.int32, device=dev)
    bits = ext.tree_bits([[-1, 0, 0, 1]] * B).to(dev)
    slots = torch.cat([torch.tensor([int(table[b, (c + j) // page]) * page + (c + j) % page for j in range(n)])
                       for b, c in enumerate(ctx.tolist())]).to(dev)
    proj = rn(N, (2 * HQ + 2 * HKV) * D).bfloat16()
    qw, kw = torch.ones(D, device=dev), torch.ones(D, device=dev)
    ang = torch.rand(N, 32, generator=g, device=dev) * 6
    cos, sin = torch.cat([ang.cos()] * 2, 1).bfloat16(), torch.cat([ang.sin()] * 2, 1).bfloat16()
    wo = (rn(256, HQ * D) * 0.02).bfloat16()
    h, w1 = rn(N, 256).bfloat16(), torch.ones(256, device=dev)
    lin = [t.to(dev) for t in _lin_case(N, 1, 3, True, seed)]
    pool = 0.1 * rn(N, 3, 128, 128)
    slot = torch.arange(N, dtype=torch.int32, device=dev)
    fill = rn(pages, HKV, page, D)
    cache[0].copy_(fill.to(torch.float8_e4m3fn))
    cache[1].copy_((fill * 0.5).to(torch.float8_e4m3fn))

    def step():
        qt, kt, vt, gate = ext.fullattn_prep2(proj, qw, kw, cos, sin, 1, N, HQ, HKV, D, 1e-6)
        ext.kv_cache_write(kt, vt, slots, *cache)
        y = ext.tree_attn(qt, cache[0], cache[1], table, ctx, q_ptr, bits, cache[2], cache[3])
        hn = ext.mm_residual_rmsnorm(h, y, wo, w1, None, 1e-6)
        p, last = ext.linattn_prompt(*lin, q_ptr, pool[:B].contiguous(), None)
        o = ext.linattn_step(*lin, pool, slot)
        k2, v2 = ext.kv_cache_read(cache[0], cache[1], slots, cache[2], cache[3])
        return [*hn, p, last, o, pool, k2, v2, qt, kt, vt, y]

    return step, dict(proj=proj, lin=lin, pool=pool, cache=cache, table=table, ctx=ctx, q_ptr=q_ptr, bits=bits)


def test_layers_run_together(ext, C, dev):
    """Prep, cache write, tree attention and out-projection; linear attention in both forms: the outputs of each against
    the oracle on what the call before gave."""
    step, t = _layers(ext, dev, 5)
    start = t["pool"].clone()
    h, hn, p, last, o, pool, k2, v2, qt, kt, vt, y = step()
    c = dict(q=qt[0].cpu(), kc=t["cache"][0].cpu(), vc=t["cache"][1].cpu(), ks=t["cache"][2].cpu(), vs=t["cache"][3].cpu(),
             table=t["table"].cpu(), ctx=t["ctx"].cpu(), q_ptr=t["q_ptr"].cpu(), bits=t["bits"].cpu())
    val, scale = C.cache_store(kt[0].cpu())
    assert torch.equal(k2.cpu().double(), (val * scale[..., None]))
    lse = ext.tree_attn(qt, t["cache"][0], t["cache"][1], t["table"], t["ctx"], t["q_ptr"], t["bits"], t["cache"][2],
                        t["cache"][3], want_lse=True)[1]
    _check_tree(C, c, y, lse, 1 / 16)
    lin = [x.cpu() for x in t["lin"]]
    _check_lin(C, lin, [4, 4, 4], start[:3].cpu(), p, last, 128 ** -0.5)
    _check_lin(C, lin, [1] * 12, start.cpu(), o, pool, 128 ** -0.5)
    assert bool(torch.isfinite(h.float()).all()) and bool(torch.isfinite(hn.float()).all())


def test_layers_in_two_graphs(ext, dev):
    """Two captured steps on inputs of their own, replayed in turn with eager work between, equal the eager calls."""
    runs = []
    for seed in (1, 2):
        step, t = _layers(ext, dev, seed)
        saved = t["pool"].clone(), [x.clone() for x in t["cache"]]

        def reset(t=t, saved=saved):
            t["pool"].copy_(saved[0])
            for x, y in zip(t["cache"], saved[1]):
                x.view(torch.uint8).copy_(y.view(torch.uint8))

        want = [x.clone() for x in step()]
        reset()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs = step()
        runs.append((graph, outs, want, reset, step))
    for r in range(4):
        for graph, outs, want, reset, step in runs:
            reset()
            graph.replay()
            torch.cuda.synchronize()
            for i, (a, b) in enumerate(zip(outs, want)):
                assert torch.equal(a, b), f"replay {r}: output {i}"
        runs[r % 2][3]()
        runs[r % 2][4]()          # eager work of the same shapes between replays
        torch.cuda.synchronize()


def test_cores_on_streams_at_once(ext, dev):
    """The same calls on two streams at once, each with its own tensors."""
    lots = []
    for seed in (3, 4):
        step, t = _layers(ext, dev, seed)
        saved = t["pool"].clone()
        want = [x.clone() for x in step()]
        t["pool"].copy_(saved)
        lots.append((step, want, torch.cuda.Stream()))
    torch.cuda.synchronize()
    got = []
    for step, want, s in lots:
        with torch.cuda.stream(s):
            got.append(step())
    torch.cuda.synchronize()
    for (step, want, s), outs in zip(lots, got):
        for i, (a, b) in enumerate(zip(outs, want)):
            assert torch.equal(a, b), f"output {i}"


def test_cores_give_the_same_bits_again(ext, dev):
    c = _tree_case([12, 30], [1000, 77], 2, 6, 256, 64, "bf16", dev, seed=8, ext=ext)
    a, b = _run_tree(ext, c, dev), _run_tree(ext, c, dev)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    args = _put(dev, *_lin_case(500, 2, 3, True, seed=8), torch.tensor([0, 100, 500], dtype=torch.int32))
    a, b = ext.linattn_prompt(*args), ext.linattn_prompt(*args)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
