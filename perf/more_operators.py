"""Performance cases of what a decoding step with drafted tokens does around its attention: linear attention over a tree of
drafted tokens, the verification of the tokens against the target's distributions, and what becomes of the caches then.

Every sequence brings a few rows to a step: its last token (row 0) and drafted ones, each with the row that it follows. The
sizes are the hybrid model's (4 key heads of 256 in 16 layers with a paged cache; 16 key and 48 value heads of 128 in the
layers with a state) and others of the same kinds for the drawn cases; vocabularies are of 1000 to 131072 tokens.

A case's "op" says what runs:
  verify  ext.verify_drafts: drafted tokens accepted or not from given random numbers, and each sequence's next token
  tree    ext.linattn_tree: linear attention of drafted trees on states that stay as they are
  state   ext.linattn_keep: states taken forward over the accepted tokens, in place
  rows    ext.kv_cache_keep: the accepted tokens' keys and values moved together, in every layer of a paged cache
  pages   ext.kv_pages_resize, kv_pages_fork, kv_pages_copy: pages freed and taken, sequences forked, their last pages copied

`own` chooses between the package's kernels and plain torch operations.
"""
import functools
import math

import torch

own = False

HD = 128     # head size of the linear-attention layers


# ------------------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one sequence, tokens looked up in its text (no draft probabilities): launch latency
        {"name": "verify_1x6", "op": "verify", "B": 1, "n": 6, "V": 32000, "pad": 0, "bits": 16, "probs": "none",
         "tree": False},
        # a few sequences with a draft model's line of tokens; fp32 logits, a vocabulary that is no multiple of anything
        {"name": "verify_16x5_odd", "op": "verify", "B": 16, "n": 5, "V": 100003, "pad": 5, "bits": 32, "probs": "bf16",
         "tree": False},
        # a full batch of trees with a draft model's probabilities: the most data
        {"name": "verify_64x12_tree", "op": "verify", "B": 64, "n": 12, "V": 131072, "pad": 0, "bits": 16, "probs": "fp32",
         "tree": True},
        # one sequence's tree: latency
        {"name": "tree_1x8", "op": "tree", "B": 1, "n": 8, "HK": 16, "G": 3, "delta": True},
        # a full batch of trees
        {"name": "tree_64x12", "op": "tree", "B": 64, "n": 12, "HK": 16, "G": 3, "delta": True},
        # wide trees of few sequences
        {"name": "tree_8x64", "op": "tree", "B": 8, "n": 64, "HK": 16, "G": 3, "delta": True},
        # one sequence goes on by up to five tokens: latency
        {"name": "state_1x5", "op": "state", "B": 1, "n": 8, "keep": 5, "HK": 16, "G": 3, "delta": True},
        # a full batch
        {"name": "state_64x6", "op": "state", "B": 64, "n": 12, "keep": 6, "HK": 16, "G": 3, "delta": True},
        # one layer of one sequence: launch latency
        {"name": "rows_1x5", "op": "rows", "B": 1, "n": 8, "keep": 5, "ctx": 539, "HKV": 4, "D": 256, "page": 64,
         "fmt": "bf16", "layers": 1},
        # all sixteen layers of a full batch, quantised
        {"name": "rows_64x6_e4m3", "op": "rows", "B": 64, "n": 12, "keep": 6, "ctx": 150, "HKV": 4, "D": 256, "page": 64,
         "fmt": "e4m3", "layers": 16},
        # one prompt's sequence answered three more times, in a single layer's cache
        {"name": "pages_1x3", "op": "pages", "P": 1, "forks": 3, "ctx": 539, "HKV": 4, "D": 256, "page": 64, "fmt": "bf16",
         "layers": 1},
        # eight prompts of up to 1000 tokens, seven more answers each, in all sixteen layers
        {"name": "pages_8x7", "op": "pages", "P": 8, "forks": 7, "ctx": 1000, "HKV": 4, "D": 256, "page": 64, "fmt": "bf16",
         "layers": 16},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("verify", "verify", "tree", "tree", "state", "rows", "pages"))
    if op == "verify":
        c = {"op": op, "B": _log_int(rng, 1, 64), "n": _log_int(rng, 1, 32), "V": _log_int(rng, 1000, 131072),
             "pad": rng.choice((0, 0, 3, 8)), "bits": rng.choice((16, 16, 32)),
             "probs": rng.choice(("none", "bf16", "fp32")), "tree": rng.random() < 0.5}
        while c["B"] * c["n"] * c["V"] * c["bits"] > 64 * 12 * 131072 * 16:
            c["V"] = max(1000, c["V"] * 2 // 3)
        return c
    heads = {"HK": rng.choice((1, 2, 4, 16, 16)), "G": rng.choice((1, 2, 3, 3)), "delta": rng.random() < 0.8}
    if op == "tree":
        c = {"op": op, "B": _log_int(rng, 1, 64), "n": _log_int(rng, 1, 64), **heads}
        while c["B"] * (c["n"] + 8) > 64 * 20:
            c["n"] = max(1, c["n"] * 2 // 3)
        return c
    n = _log_int(rng, 1, 32)
    if op == "state":
        return {"op": op, "B": _log_int(rng, 1, 64), "n": n, "keep": rng.randint(1, min(n, 12)), **heads}
    cache = {"HKV": rng.choice((1, 2, 4, 8)), "D": rng.choice((128, 256, 256)), "page": rng.choice((16, 32, 64, 128)),
             "fmt": rng.choice(("e4m3", "bf16")), "layers": rng.choice((1, 2, 5, 16))}
    if op == "rows":
        c = {"op": op, "B": _log_int(rng, 1, 64), "n": n, "keep": rng.randint(1, min(n, 12)), "ctx": _log_int(rng, 1, 400),
             **cache}
        size = lambda: c["B"] * (c["ctx"] + c["n"] + c["page"]) * c["HKV"] * c["D"] * c["layers"]  # noqa: E731
        while size() > 64 * 226 * 4 * 256 * 16:
            c["layers"], c["B"] = max(1, c["layers"] // 2), max(1, c["B"] * 2 // 3)
        return c
    c = {"op": op, "P": _log_int(rng, 1, 16), "forks": rng.randint(1, 8), "ctx": _log_int(rng, 1, 1000), **cache}
    size = lambda: c["P"] * (c["ctx"] + c["forks"] * c["page"]) * c["HKV"] * c["D"] * c["layers"]  # noqa: E731
    while size() > 8 * (1000 + 7 * 64) * 4 * 256 * 16:
        c["layers"], c["P"] = max(1, c["layers"] // 2), max(1, c["P"] * 2 // 3)
    return c


def _lengths(count, most, least):
    """Lengths of `count` sequences: the first the longest, the others spread between least and most."""
    return [most] + [least + int((most - least) * ((i * 0.6180339887) % 1.0)) for i in range(1, count)]


def _rows(c):
    """Rows of each sequence; of four or more, one has none."""
    n = _lengths(c["B"], c["n"], (c["n"] + 1) // 2)
    if c["B"] >= 4:
        n[2] = 0
    return n


def _kept(c):
    """Accepted tokens of each sequence, its last token among them."""
    return [min(a, b) for a, b in zip(_lengths(c["B"], c["keep"], 1), _rows(c))]


def _contexts(c):
    """Cached tokens of each prompt's sequence, or of each sequence."""
    count = c["P"] if c["op"] == "pages" else c["B"]
    return _lengths(count, c["ctx"], (c["ctx"] + 3) // 4)


def _follows(c, seed):
    """The row that each row follows, -1 for a sequence's row 0: the one before it, or of a tree one of the six before it."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for n in _rows(c):
        pick = torch.rand(n, generator=g).tolist()
        out += [-1 if j == 0 else (j - 1 if not c.get("tree", True) else max(0, j - 6) + int(pick[j] * min(j, 6)))
                for j in range(n)]
    return out


def _paths(c, seed):
    """Accepted rows of each sequence: row 0, then rising ones."""
    g = torch.Generator().manual_seed(seed)
    return [[0] + sorted((1 + torch.randperm(n - 1, generator=g)[:m - 1]).tolist()) if m else []
            for n, m in zip(_rows(c), _kept(c))]


def work(c):
    """What the outputs cannot do without. Verification: every logit once (any row may turn out to be the last), of the
    draft's probabilities those of the drafted tokens. Rows: those that move, about all but each sequence's first."""
    if c["op"] == "verify":
        N = sum(_rows(c))
        return {"bytes": N * c["V"] * c["bits"] // 8 + N * 24 + c["B"] * 16, "flops": 4 * N * c["V"]}
    if c["op"] in ("tree", "state"):
        n = _rows(c) if c["op"] == "tree" else _kept(c)
        HK, HV = c["HK"], c["HK"] * c["G"]
        wide = (2, 2) if c["op"] == "tree" else (1, 1)       # q and o too
        token = (wide[0] * HK * HD + wide[1] * HV * HD) * 2 + HV * (4 + (2 if c["delta"] else 0))
        live = sum(1 for x in n if x)
        reads = 1 if c["op"] == "tree" else 2
        flops = (4 if c["op"] == "tree" else 2) + (2 if c["op"] == "state" and c["delta"] else 0)
        return {"bytes": live * reads * HV * HD * HD * 4 + sum(n) * token, "flops": sum(n) * flops * HD * HD * HV}
    e = 1 if c["fmt"] == "e4m3" else 2
    token = c["layers"] * c["HKV"] * (2 * c["D"] * e + (8 if e == 1 else 0))
    if c["op"] == "rows":
        return {"bytes": 2 * token * sum(max(0, m - 1) for m in _kept(c)), "flops": 0}
    last = sum(x % c["page"] for x in _contexts(c))          # tokens in last pages
    return {"bytes": 2 * token * last * c["forks"], "flops": 0}


# --------------------------------------------------------------------------------------------------------------- inputs
class _Rand:
    """Draws on the GPU from one seed."""

    def __init__(self, seed):
        self.dev = torch.device("cuda")
        self.g = torch.Generator(device=self.dev)
        self.g.manual_seed(seed)

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.g, device=self.dev)

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.g, device=self.dev)

    def perm(self, n):
        return torch.randperm(n, generator=self.g, device=self.dev)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _pointers(lengths):
    at = [0]
    for x in lengths:
        at.append(at[-1] + x)
    return _ints(at)


def _pool(r, c, pages):
    """kc, vc, ks, vs of a cache of all layers that holds keys and values."""
    shape = (c["layers"], pages, c["HKV"], c["page"], c["D"])
    kc, vc = torch.empty(shape, dtype=torch.bfloat16, device="cuda"), torch.empty(shape, dtype=torch.bfloat16, device="cuda")
    for x in (kc, vc):
        x.normal_(generator=r.g)
    if c["fmt"] == "bf16":
        return kc, vc, None, None
    # quantised with a scale for each token and head
    sc = [torch.exp2(torch.floor(3 * r.uniform(*shape[:4])) - 9) for _ in range(2)]
    return (kc * 64).to(torch.float8_e4m3fn), (vc * 64).to(torch.float8_e4m3fn), sc[0], sc[1]


def _verify_state(c, r, seed):
    n, V = _rows(c), c["V"]
    N, B = sum(n), c["B"]
    dtype = torch.bfloat16 if c["bits"] == 16 else torch.float32
    # a dozen tokens far above the rest, as a language model has them
    raw = 2.0 * r.normal(N, V + c["pad"])
    high = (r.uniform(N, 12) * V).long()
    raw.scatter_(1, high, 6.0 + 8.0 * r.uniform(N, 12))
    logits = raw.to(dtype)[:, :V]                       # rows of a projection whose width is a multiple of its own
    temp = _ints([(0.8, 1.0, 0.6, 0.0)[b % 4] for b in range(B)], torch.float32)
    owner = torch.repeat_interleave(torch.arange(B, device="cuda"), _ints(n, torch.int64))
    parents, ptr = _ints(_follows(c, seed)), _pointers(n)
    above = ptr[owner].long() + parents.long().clamp_min(0)
    # the draft's own distributions, near the target's, and its tokens drawn from the row that each of them follows
    draft = raw[:, :V].mul_(0.9)
    draft += 0.5 * r.normal(N, V)
    draft = torch.softmax(draft / temp[owner].clamp_min(0.3)[:, None], -1)
    sums = draft.cumsum(-1)
    tokens = torch.searchsorted(sums[above], r.uniform(N, 1) * sums[above, -1:])[:, 0].clamp_max(V - 1)
    probs = {"none": None, "bf16": draft.bfloat16(), "fp32": draft}[c["probs"]]
    return {"c": c, "logits": logits, "tokens": tokens, "q_ptr": ptr, "u": r.uniform(N), "probs": probs,
            "parents": parents if c["tree"] else None, "temperature": temp}


def prepare(c, seed):
    r = _Rand(seed)
    if c["op"] == "verify":
        return _verify_state(c, r, seed)
    if c["op"] in ("tree", "state"):
        HK, HV = c["HK"], c["HK"] * c["G"]
        n, B = _rows(c), c["B"]
        R = sum(n)
        qk = torch.nn.functional.silu(r.normal(2, R, HK, HD) + 0.3)
        q, k = (qk / (qk.square().sum(-1, keepdim=True) + 1e-6).sqrt()).bfloat16().reshape(2, R, HK * HD)
        v = torch.nn.functional.silu(r.normal(R, HV * HD)).bfloat16()
        decay = 1.0 + 15.0 * r.uniform(HV)                                    # exp(A_log)
        step = torch.exp(r.uniform(HV) * math.log(100.0) + math.log(1e-3))    # softplus(dt_bias), 0.001 .. 0.1
        bias = step + torch.log(-torch.expm1(-step))
        g = -decay * torch.nn.functional.softplus(r.normal(R, HV) + bias)
        s = {"c": c, "k": k.contiguous(), "v": v, "g": g, "q_ptr": _pointers(n),
             "beta": torch.sigmoid(r.normal(R, HV)).bfloat16() if c["delta"] else None,
             "state": 0.1 * r.normal(B + 2, HV, HD, HD), "slot": r.perm(B + 2)[:B].int()}
        if c["op"] == "tree":
            return {**s, "q": q.contiguous(), "parents": _ints(_follows(c, seed)), "scale": HD ** -0.5}
        paths = _paths(c, seed)
        s["path"] = _ints([x for p, m in zip(paths, n) for x in p + [-1] * (m - len(p))])
        s["count"] = _ints([len(p) for p in paths])
        return s
    PS, ctx = c["page"], _contexts(c)
    if c["op"] == "rows":
        n, B = _rows(c), c["B"]
        need = [-(-(x + y) // PS) for x, y in zip(n, ctx)]
        pages = sum(need) + 2
        order, at = r.perm(pages).int(), 0
        table = torch.full((B, max(need)), -1, dtype=torch.int32, device="cuda")
        for b in range(B):
            table[b, :need[b]] = order[at:at + need[b]]
            at += need[b]
        paths = _paths(c, seed)
        kc, vc, ks, vs = _pool(r, c, pages)
        return {"c": c, "kc": kc, "vc": vc, "ks": ks, "vs": vs, "table": table, "ctx": _ints(ctx), "q_ptr": _pointers(n),
                "path": _ints([x for p, m in zip(paths, n) for x in p + [-1] * (m - len(p))]),
                "count": _ints([len(p) for p in paths])}
    # pages: prompts in slots 0 .. P - 1, empty slots for their forks; every fifth page belongs to sequences elsewhere
    P, F = c["P"], c["forks"]
    B, need = P * (1 + F), [-(-x // PS) for x in ctx]
    used = sum(need)
    pages = (used + P * F) * 5 // 4 + 8
    order = r.perm(pages).int()
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    table = torch.full((B, max(need) + 1), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b in range(P):
        table[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
    refs[order[:used + pages // 5].long()] = 1
    kc, vc, ks, vs = _pool(r, c, pages)
    return {"c": c, "kc": kc, "vc": vc, "ks": ks, "vs": vs, "table": table, "refs": refs,
            "ctx": _ints(ctx + [0] * (P * F)), "tokens": _ints([-1] * P + [0] * (P * F)),
            "src": _ints(list(range(P)) + [b % P for b in range(P * F)])}


# ---------------------------------------------------------------------------------------------------------- plain forms
def _padded(s, first, lengths, most):
    """Row numbers of the sequences side by side [B, most], and which of them are there."""
    i = torch.arange(most, device="cuda")
    live = i[None] < lengths[:, None]
    return torch.where(live, first[:, None] + i[None], 0), live


def _distributions(logits, temp):
    """softmax(logits / temp) in 64 bits; all on the first largest where the temperature is 0."""
    x = logits.double()
    top = x.amax(-1, keepdim=True)
    e = torch.exp((x - top) / torch.where(temp > 0, temp, 1.0)[:, None])
    first = torch.nn.functional.one_hot(x.argmax(-1), x.shape[1]).double()
    return torch.where((temp > 0)[:, None], e / e.sum(-1, keepdim=True), first)


def _verify_plain(s):
    c, V, dev = s["c"], s["c"]["V"], s["logits"].device
    ptr = s["q_ptr"].long()
    first, lengths = ptr[:-1], ptr[1:] - ptr[:-1]
    B, N, most = c["B"], s["logits"].shape[0], c["n"]
    row, live = _padded(s, first, lengths, most)
    temp = s["temperature"].double()
    # without a tree each row follows the one before it
    parents = s["parents"].long()[row] if s["parents"] is not None else torch.arange(-1, most - 1, device=dev).expand(B, -1)
    b = torch.arange(B, device=dev)
    last = max(0, N - 1)
    cur = torch.zeros(B, dtype=torch.long, device=dev)
    left = _distributions(s["logits"][first.clamp_max(last)], temp)
    total, shift = torch.ones(B, dtype=torch.float64, device=dev), torch.zeros(B, dtype=torch.float64, device=dev)
    path = torch.full((B, most), -1, dtype=torch.int32, device=dev)
    path[:, 0] = 0
    count = torch.ones(B, dtype=torch.long, device=dev)
    for j in range(1, most):
        x, tested = s["tokens"][row[:, j]], live[:, j] & (parents[:, j] == cur)
        node = (first + cur).clamp_max(last)
        q = torch.ones_like(total) if s["probs"] is None else s["probs"][node, x].double()
        q = torch.where(temp > 0, q, 1.0)
        yes = tested & (s["u"][row[:, j]].double() * q * total < left[b, x])
        no = tested & ~yes & (temp > 0)
        if s["probs"] is None:
            less = left.scatter(1, x[:, None], 0.0)
        else:
            shift = torch.where(no, shift + total, torch.where(yes, 0.0, shift))
            less = (_distributions(s["logits"][node], temp) - shift[:, None] * s["probs"][node].double()).clamp_min(0)
        left = torch.where(no[:, None], less, left)
        left = torch.where(yes[:, None], _distributions(s["logits"][row[:, j]], temp), left)
        total = torch.where(no, left.sum(-1), torch.where(yes, 1.0, total))
        path[b, torch.where(yes, count, 0)] = torch.where(yes, j, 0).int()
        count = count + yes
        cur = torch.where(yes, j, cur)
    left = torch.where((total > 0)[:, None], left, _distributions(s["logits"][(first + cur).clamp_max(last)], temp))
    sums = left.cumsum(-1)
    u = torch.where(temp > 0, s["u"][first.clamp_max(last)].double(), 0.0)
    token = (sums <= (u * sums[:, -1])[:, None]).sum(-1)
    some = lengths > 0
    out = torch.full((N,), -1, dtype=torch.int32, device=dev)
    out[row[live]] = path[live]
    return [out, torch.where(some, count, 0).int(), torch.where(some, token, -1)]


def _unit_lower_inverse(A):
    """(I + A)^-1 of strictly lower A [.., C, C]: inverses of blocks joined two by two."""
    C = A.shape[-1]
    at = torch.arange(C, device=A.device)
    T = torch.eye(C, device=A.device, dtype=A.dtype).expand(A.shape)
    size = 1
    while size < C:
        odd, pair = at // size % 2, at // (2 * size)
        join = (odd[:, None] == 1) & (odd[None] == 0) & (pair[:, None] == pair[None])
        T = T - T @ (A * join) @ T
        size *= 2
    return T


def _tree_plain(s):
    c = s["c"]
    B, HK, HV, C = c["B"], c["HK"], c["HK"] * c["G"], c["n"]
    ptr, dev = s["q_ptr"].long(), s["q"].device
    row, live = _padded(s, ptr[:-1], ptr[1:] - ptr[:-1], C)
    parents = torch.where(live, s["parents"].long()[row], -1)
    # ancestors and self: the closure of "follows" by squaring
    seen = (parents[..., None] == torch.arange(C, device=dev)).float() + torch.eye(C, device=dev)
    for _ in range(max(1, (C - 1).bit_length())):
        seen = (seen @ seen).clamp_max(1.0)
    seen = (seen > 0)[:, None]                                                      # [B, 1, C, C]

    def laid(x, heads):   # [R, heads * w] -> fp32 [B, HV, C, w], zeros behind a sequence's end
        x = torch.where(live[..., None, None], x.float().reshape(x.shape[0], heads, -1)[row], 0.0)
        return x.transpose(1, 2).repeat_interleave(HV // heads, 1)

    q, k, v = laid(s["q"], HK), laid(s["k"], HK), laid(s["v"], HV)
    sums = (seen.double() @ laid(s["g"], HV).double())[..., 0]                      # [B, HV, C]
    fade = torch.where(seen, sums[..., :, None] - sums[..., None, :], -math.inf).exp().float()
    since = sums.exp().float()[..., None]
    state = s["state"][s["slot"].long()]
    u = v
    if c["delta"]:
        beta = laid(s["beta"], HV)
        A = (beta * (fade * (k @ k.transpose(-1, -2)))).tril(-1)
        u = _unit_lower_inverse(A) @ (beta * (v - since * (k @ state)))
    o = s["scale"] * (since * (q @ state) + (fade * (q @ k.transpose(-1, -2))) @ u)
    return [o.transpose(1, 2)[live].reshape(-1, HV * HD).bfloat16()]


def _state_plain(s):
    c = s["c"]
    HK, HV = c["HK"], c["HK"] * c["G"]
    first, slot = s["q_ptr"][:-1].long(), s["slot"].long()
    state = s["state"][slot]
    for i in range(c["keep"]):
        on = i < s["count"].long()
        at = torch.where(on, first + i, 0)
        row = torch.where(on, first + s["path"].long()[at].clamp_min(0), 0)
        k = s["k"][row].float().reshape(-1, HK, HD).repeat_interleave(c["G"], 1)
        u = s["v"][row].float().reshape(-1, HV, HD)
        new = state * s["g"][row].exp()[..., None, None]
        if c["delta"]:
            u = s["beta"][row].float()[..., None] * (u - (k[..., None, :] @ new)[..., 0, :])
        state = torch.where(on[:, None, None, None], new + k[..., :, None] * u[..., None, :], state)
    s["state"][slot] = state
    return [s["state"]]


def _bytes(s):
    return [t.view(torch.uint8) if t.dtype is torch.float8_e4m3fn else t
            for t in (s["kc"], s["vc"], s["ks"], s["vs"]) if t is not None]


def _cache(s):
    return [t for t in (s["kc"], s["vc"], s["ks"], s["vs"]) if t is not None]


def _rows_plain(s):
    PS, keep = s["c"]["page"], s["c"]["keep"]
    row, _ = _padded(s, s["q_ptr"][:-1].long(), s["count"].long(), keep)
    i = torch.arange(keep, device="cuda")[None]
    on = i < s["count"].long()[:, None]
    path = torch.where(on, s["path"].long()[row], i)
    ctx = s["ctx"].long()[:, None]
    width = s["table"].shape[1] * PS

    def place(pos):
        pos = pos.clamp_max(width - 1)
        return torch.gather(s["table"].long(), 1, pos // PS), pos % PS

    (fp, fo), (tp, to) = place(ctx + path), place(ctx + i + 0 * path)
    # what does not move is written where it lies; a sequence's places behind its kept rows are not touched
    moved = on & (path != i)
    for t in _bytes(s):
        x = t[:, fp[moved], :, fo[moved]]                  # read before anything is written
        t[:, tp[moved], :, to[moved]] = x
    return _cache(s)


def _pages_plain(s):
    table, refs, ctx, PS = s["table"], s["refs"], s["ctx"], s["c"]["page"]
    B, MP = table.shape
    pages, i = refs.shape[0], torch.arange(MP, device="cuda")

    def there(t):
        return (t >= 0) & (t < pages)

    def counted(t, one):
        """refs + one for each entry of t that names a page."""
        ok = there(t)
        return refs.scatter_add_(0, torch.where(ok, t, 0).reshape(-1).long(), torch.where(ok, one, 0).reshape(-1).int())

    def take(wanted):
        """The lowest free pages for the entries that want one, in order, -1 where none is left; counted."""
        free = refs <= 0
        order = torch.sort((~free).int(), stable=True)[1]          # free pages first, each kind from the lowest
        rank = wanted.reshape(-1).int().cumsum(0).reshape(wanted.shape) - 1
        page = torch.where(wanted & (rank < free.sum()), order[rank.clamp(0, pages - 1)], -1).int()
        counted(page, 1)
        return page

    # resize: entries behind what a sequence wants are given back, those that it lacks are taken
    want = torch.where(s["tokens"] >= 0, (s["tokens"] + PS - 1) // PS, -1)[:, None]
    back = there(table) & (want >= 0) & (i[None] >= want)
    counted(torch.where(back, table, -1), -1)
    lacks = (i[None] < want) & ~there(table)
    table.copy_(torch.where((want >= 0) & (i[None] >= want), -1, table))
    table.copy_(torch.where(lacks, take(lacks), table))
    short = (lacks & (table < 0)).sum(-1).int()
    # fork: slots that name another slot go on as its sequence
    src, old, length = s["src"].long(), table.clone(), ctx.clone()
    b = torch.arange(B, device="cuda")
    other = src != b
    counted(torch.where(other[:, None], old, -1), -1)
    full = (length[src] // PS)[:, None]
    new = torch.where(other[:, None], torch.where(i[None] < full, old[src], -1), old)
    counted(torch.where(other[:, None], new, -1), 1)
    part = other & (length[src] % PS > 0) & (full[:, 0] < MP)
    column = full[:, 0].clamp_max(MP - 1)
    page = take(part)
    got = part & (page >= 0)
    new[b, column.long()] = torch.where(got, page, new[b, column.long()])
    pairs = torch.stack([torch.where(part, old[src, column.long()], -1), page], 1).int()
    table.copy_(new)
    ctx.copy_(torch.where(part & ~got, full[:, 0] * PS, length[src]))
    # copy: the last pages, in every layer
    at = got.nonzero()[:, 0]
    for t in _bytes(s):
        t[:, pairs[at, 1].long()] = t[:, pairs[at, 0].long()]
    return [table, refs, ctx, short, pairs] + _cache(s)


# ------------------------------------------------------------------------------------------------------------- one pass
@functools.lru_cache(None)
def _package():
    from __graft_entry__ import load_package
    load_package()
    from open_jev_fast_amd import ext
    return ext


def run(s):
    op = s["c"]["op"]
    if not own:
        return {"verify": _verify_plain, "tree": _tree_plain, "state": _state_plain, "rows": _rows_plain,
                "pages": _pages_plain}[op](s)
    ext = _package()
    if op == "verify":
        return list(ext.verify_drafts(s["logits"], s["tokens"], s["q_ptr"], s["u"], s["parents"], s["probs"],
                                      s["temperature"]))
    if op == "tree":
        return [ext.linattn_tree(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"], s["slot"], s["q_ptr"],
                                 s["parents"], scale=s["scale"])]
    if op == "state":
        ext.linattn_keep(s["k"], s["v"], s["g"], s["beta"], s["state"], s["slot"], s["q_ptr"], s["path"], s["count"])
        return [s["state"]]
    if op == "rows":
        ext.kv_cache_keep(s["kc"], s["vc"], s["table"], s["ctx"], s["q_ptr"], s["path"], s["count"], s["ks"], s["vs"])
        return _cache(s)
    short = ext.kv_pages_resize(s["table"], s["refs"], s["tokens"], s["c"]["page"])
    pairs = ext.kv_pages_fork(s["table"], s["ctx"], s["refs"], s["src"], s["c"]["page"])
    ext.kv_pages_copy(s["kc"], s["vc"], pairs, s["ks"], s["vs"])
    return [s["table"], s["refs"], s["ctx"], short, pairs] + _cache(s)


# ------------------------------------------------------------------------------------------------- the same in 64 bits
def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "verify":
        return _exact_verify(s)
    if c["op"] == "tree":
        return _exact_tree(s)
    if c["op"] == "state":
        return _exact_state(s)
    return None          # whole numbers and copies


def _exact_verify(s):
    """Sequence by sequence, child by child, each rejection's distribution made from the one before it."""
    n, c = _rows(s["c"]), s["c"]
    ptr, follows = s["q_ptr"].tolist(), None if s["parents"] is None else s["parents"].tolist()
    tokens, u, temp = s["tokens"].tolist(), s["u"].double().tolist(), s["temperature"].double().tolist()
    path, counts, nexts = [], [], []

    def target(r, t):
        x = s["logits"][r].double()
        if t <= 0:
            p = torch.zeros_like(x)
            p[(x == x.max()).nonzero()[0, 0]] = 1.0
            return p
        return torch.softmax(x / t, 0)

    for b in range(c["B"]):
        if n[b] == 0:
            counts.append(0)
            nexts.append(-1)
            continue
        first, cur, taken = ptr[b], 0, [0]
        p = target(first, temp[b])
        while True:
            at = None
            for j in range(cur + 1, n[b]):
                above = j - 1 if follows is None else follows[first + j]
                if above != cur:
                    continue
                x = tokens[first + j]
                q = s["probs"][first + cur].double() if s["probs"] is not None and temp[b] > 0 else None
                qx = 1.0 if q is None else q[x].item()
                if u[first + j] * qx < p[x].item():
                    at = j
                    break
                if q is None:
                    rest = p.clone()
                    rest[x] = 0.0
                else:
                    rest = (p - q).clamp_min(0)
                total = rest.sum()
                p = rest / total if total > 0 else p
            if at is None:
                break
            cur = at
            taken.append(at)
            p = target(first + cur, temp[b])
        sums = p.cumsum(0)
        level = (u[first] if temp[b] > 0 else 0.0) * sums[-1].item()
        nexts.append(int((sums > level).nonzero()[0, 0]))
        path += taken + [-1] * (n[b] - len(taken))
        counts.append(len(taken))
    return [_ints(path), _ints(counts), _ints(nexts, torch.int64)]


def _one_token(state, k, v, g, beta):
    """state [HV, 128, 128] after a token, in 64 bits."""
    state = state * g.exp()[:, None, None]
    if beta is not None:
        v = beta[:, None] * (v - torch.matmul(k[:, None, :], state)[:, 0])
    return state + k[:, :, None] * v[:, None, :]


def _heads(s, r):
    c = s["c"]
    HK, HV = c["HK"], c["HK"] * c["G"]
    k = s["k"][r].double().reshape(HK, HD).repeat_interleave(c["G"], 0)
    return k, s["v"][r].double().reshape(HV, HD), s["g"][r].double(), None if s["beta"] is None else s["beta"][r].double()


def _exact_tree(s):
    """Every row's state from the state of the row that it follows."""
    c = s["c"]
    follows, ptr, slot = s["parents"].tolist(), s["q_ptr"].tolist(), s["slot"].tolist()
    out = torch.zeros(ptr[-1], c["HK"] * c["G"], HD, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_rows(c)):
        states = []
        for j in range(n):
            r = ptr[b] + j
            before = states[follows[r]] if follows[r] >= 0 else s["state"][slot[b]].double()
            states.append(_one_token(before, *_heads(s, r)))
            q = s["q"][r].double().reshape(c["HK"], HD).repeat_interleave(c["G"], 0)
            out[r] = s["scale"] * torch.matmul(q[:, None, :], states[j])[:, 0]
    return [out.reshape(ptr[-1], -1)]


def _exact_state(s):
    c = s["c"]
    ptr, slot, path, count = (s[x].tolist() for x in ("q_ptr", "slot", "path", "count"))
    held = s["state"].double()
    for b in range(c["B"]):
        for i in range(count[b]):
            held[slot[b]] = _one_token(held[slot[b]], *_heads(s, ptr[b] + path[ptr[b] + i]))
    return [held]
