"""Performance cases of the two attention cores and of the cache that one of them reads.

The hybrid model has two kinds of layers. A full-attention layer writes its keys and values to a paged cache, in bf16 or
quantised to e4m3 with a scale for each token and head, and attends from one or more drafted tokens of every sequence (a
tree of them, or a plain continuation) over the cache. A linear-attention layer carries a state of 128 x 128 for each value
head: prompts run through it in chunks, single tokens one step at a time. The sizes are the model's (24 query and 4 key
heads of 256; 16 key and 48 value heads of 128), and others of the same kinds for the drawn cases.

A case's "op" says what runs:
  write   ext.kv_cache_write: N tokens' keys and values to their slots of a paged cache
  read    ext.kv_cache_read: N tokens' keys and values from their slots, as bf16
  tree    ext.tree_attn: attention of drafted tokens over a paged cache
  prompt  ext.linattn_prompt: linear attention over whole sequences
  step    ext.linattn_step: linear attention, one token for each row, the states updated in place

`own` chooses between the package's kernels and plain torch operations.
"""
import functools
import math

import torch

own = False

HD = 128     # head size of the linear-attention layers
CHUNK = 64   # tokens taken together by the plain form of a prompt


# ------------------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # a decoding batch's new tokens, one for each sequence: launch latency
        {"name": "write_64_e4m3", "op": "write", "N": 64, "HKV": 4, "D": 256, "page": 64, "fmt": "e4m3"},
        # the longest prompt that the server takes, written in one go
        {"name": "write_16384_e4m3", "op": "write", "N": 16384, "HKV": 4, "D": 256, "page": 64, "fmt": "e4m3"},
        # a request's shared text read back for the packed forward, no multiple of a page
        {"name": "read_539_e4m3", "op": "read", "N": 539, "HKV": 4, "D": 256, "page": 64, "fmt": "e4m3"},
        # the longest prompt read back
        {"name": "read_16384_e4m3", "op": "read", "N": 16384, "HKV": 4, "D": 256, "page": 64, "fmt": "e4m3"},
        # one sequence, one token, a short text: latency
        {"name": "tree_1x1_ctx539", "op": "tree", "B": 1, "n": 1, "ctx": 539, "HKV": 4, "G": 6, "D": 256, "page": 64,
         "fmt": "bf16", "tree": False},
        # a batch of sequences with a dozen drafted tokens each over a quantised cache
        {"name": "tree_16x12_ctx8192_e4m3", "op": "tree", "B": 16, "n": 12, "ctx": 8192, "HKV": 4, "G": 6, "D": 256,
         "page": 64, "fmt": "e4m3", "tree": True},
        # wide trees over long contexts: the largest products of the section
        {"name": "tree_4x64_ctx16384", "op": "tree", "B": 4, "n": 64, "ctx": 16384, "HKV": 4, "G": 6, "D": 256, "page": 64,
         "fmt": "bf16", "tree": True},
        # the example request as one sequence
        {"name": "prompt_1x288", "op": "prompt", "S": 1, "L": 288, "HK": 16, "G": 3, "delta": True, "state": False},
        # candidate paths of a request that go on from states of their own, ragged
        {"name": "prompt_16x539", "op": "prompt", "S": 16, "L": 539, "HK": 16, "G": 3, "delta": True, "state": True},
        # the longest prompt: a long chain of chunks
        {"name": "prompt_1x16384", "op": "prompt", "S": 1, "L": 16384, "HK": 16, "G": 3, "delta": True, "state": False},
        # one sequence being decoded: latency
        {"name": "step_1", "op": "step", "B": 1, "HK": 16, "G": 3, "delta": True},
        # a decoding batch: states read and written once
        {"name": "step_64", "op": "step", "B": 64, "HK": 16, "G": 3, "delta": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("write", "read", "tree", "tree", "prompt", "prompt", "step"))
    page, fmt = rng.choice((16, 32, 64, 128)), rng.choice(("e4m3", "e4m3", "bf16"))
    D = rng.choice((128, 256, 256))
    if op in ("write", "read"):
        return {"op": op, "N": _log_int(rng, 1, 16384), "HKV": rng.choice((1, 2, 4, 8)), "D": D, "page": page, "fmt": fmt}
    if op == "tree":
        c = {"op": op, "B": _log_int(rng, 1, 32), "n": _log_int(rng, 1, 128), "ctx": _log_int(rng, 1, 16384),
             "HKV": rng.choice((1, 2, 4)), "G": rng.choice((1, 2, 3, 4, 6, 8)), "D": D, "page": page, "fmt": fmt,
             "tree": rng.random() < 0.7}
        while c["B"] * (c["n"] + 16) * (c["ctx"] + 256) * c["HKV"] * c["G"] > 4 * 64 * 16384 * 24:
            c["ctx"] = max(1, c["ctx"] * 2 // 3)
        return c
    heads = {"HK": rng.choice((1, 2, 4, 16, 16)), "G": rng.choice((1, 2, 3, 3)), "delta": rng.random() < 0.8}
    if op == "prompt":
        S = _log_int(rng, 1, 32)
        return {"op": op, "S": S, "L": _log_int(rng, 1, 16384 // S), **heads, "state": rng.random() < 0.5}
    return {"op": op, "B": _log_int(rng, 1, 128), **heads}


def _lengths(count, most, least):
    """Lengths of `count` sequences: the first the longest, the others spread between least and most."""
    return [most] + [least + int((most - least) * ((i * 0.6180339887) % 1.0)) for i in range(1, count)]


def _tree_lengths(c):
    """Drafted and cached tokens of each sequence. Of four or more, one has drafted nothing and one has nothing cached."""
    n, ctx = _lengths(c["B"], c["n"], (c["n"] + 1) // 2), _lengths(c["B"], c["ctx"], c["ctx"] // 4)
    if c["B"] >= 4:
        n[2], ctx[3] = 0, 0
    return n, ctx


def _prompt_lengths(c):
    """Sequence lengths; of four or more, one is empty."""
    L = _lengths(c["S"], c["L"], c["L"] // 3)
    if c["S"] >= 4:
        L[2] = 0
    return L


def work(c):
    e = 1 if c.get("fmt") == "e4m3" else 2
    if c["op"] in ("write", "read"):
        values = 2 * c["N"] * c["HKV"] * c["D"]
        scales = 8 * c["N"] * c["HKV"] if e == 1 else 0
        return {"bytes": values * (2 + e) + scales + 8 * c["N"], "flops": 0}
    if c["op"] == "tree":
        n, ctx = _tree_lengths(c)
        HQ, D = c["HKV"] * c["G"], c["D"]
        tokens = sum(x + y for x, y in zip(n, ctx) if x)
        cache = tokens * c["HKV"] * (2 * D * e + (8 if e == 1 else 0))
        return {"bytes": cache + sum(n) * HQ * D * 4, "flops": 4 * D * HQ * sum(x * (x + y) for x, y in zip(n, ctx))}
    HK, HV = c["HK"], c["HK"] * c["G"]
    token = (2 * HK * HD + 2 * HV * HD) * 2 + HV * (4 + (2 if c["delta"] else 0))
    states = HV * HD * HD * 4
    flops = (6 if c["delta"] else 4) * HD * HD * HV
    if c["op"] == "prompt":
        R = sum(_prompt_lengths(c))
        return {"bytes": R * token + c["S"] * states * (2 if c["state"] else 1), "flops": R * flops}
    return {"bytes": c["B"] * (token + 2 * states), "flops": c["B"] * flops}


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


def _keys_values(r, *shape):
    """Keys as they leave the norm and the rotation, and values with a few loud channels; bf16."""
    loud = 1.0 + 7.0 * (r.uniform(shape[-1]) > 0.97)
    return r.normal(*shape).bfloat16(), (0.5 * r.normal(*shape) * loud).bfloat16()


def _quantised(x):
    """e4m3 values and the scale of each row of x: the smallest power of two that brings the row within +-448."""
    x = x.float()
    m, e = torch.frexp(x.abs().amax(-1))          # amax = m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(m > 0.875, e - 8, e - 9).clamp_min(-126)
    e = torch.where(m == 0, torch.zeros_like(e), e)
    scale = torch.ldexp(torch.ones_like(m), e)
    return torch.ldexp(x, -e[..., None]).to(torch.float8_e4m3fn), scale


def _stored(k, v, fmt):
    """kc, vc, ks, vs of a cache that holds k and v."""
    if fmt == "bf16":
        return k, v, None, None
    (kc, ks), (vc, vs) = _quantised(k), _quantised(v)
    return kc, vc, ks, vs


def prepare(c, seed):
    r = _Rand(seed)
    if c["op"] in ("write", "read"):
        N, HKV, D, PS = c["N"], c["HKV"], c["D"], c["page"]
        pages = -(-N // PS) + 2
        # a sequence's tokens lie one after the other in pages from all over the pool
        at = torch.arange(N, device="cuda")
        slots = r.perm(pages)[at // PS] * PS + at % PS
        k, v = _keys_values(r, HKV, N, D)
        pool = _keys_values(r, pages, HKV, PS, D)
        kc, vc, ks, vs = _stored(*pool, c["fmt"])
        return {"c": c, "k": k, "v": v, "slots": slots, "kc": kc, "vc": vc, "ks": ks, "vs": vs}
    if c["op"] == "tree":
        B, HKV, D, PS = c["B"], c["HKV"], c["D"], c["page"]
        HQ = HKV * c["G"]
        n, ctx = _tree_lengths(c)
        need = [-(-(x + y) // PS) for x, y in zip(n, ctx)]
        pages = sum(need) + 2
        order = r.perm(pages).int()
        table = torch.full((B, max(need)), -1, dtype=torch.int32, device="cuda")
        at = 0
        for b in range(B):
            table[b, :need[b]] = order[at:at + need[b]]
            at += need[b]
        kc, vc, ks, vs = _stored(*_keys_values(r, pages, HKV, PS, D), c["fmt"])
        q = r.normal(HQ, sum(n), D).bfloat16()
        bits = None
        if c["tree"]:
            # a drafted token follows one of those drafted before it, or the context itself
            words, rows, pick = max(1, -(-max(n) // 64)), [], r.uniform(sum(n)).tolist()
            for x in n:
                seen = []
                for i in range(x):
                    parent = int(pick[len(rows)] * (min(i, 6) + 1)) + max(0, i - 6) - 1
                    seen.append((seen[parent] if parent >= 0 else 0) | 1 << i)
                    rows.append(seen[-1])
            wrap = [[(y >> 64 * w & (1 << 64) - 1) for w in range(words)] for y in rows]
            bits = _ints([[y - (1 << 64) if y >> 63 else y for y in w] for w in wrap], torch.int64)
        return {"c": c, "q": q, "kc": kc, "vc": vc, "ks": ks, "vs": vs, "table": table, "ctx": _ints(ctx),
                "q_ptr": _pointers(n), "bits": bits, "scale": D ** -0.5}
    HK, HV = c["HK"], c["HK"] * c["G"]
    L = _prompt_lengths(c) if c["op"] == "prompt" else [1] * c["B"]
    R, S = sum(L), len(L)
    qk = torch.nn.functional.silu(r.normal(2, R, HK, HD) + 0.3)
    q, k = (qk / (qk.square().sum(-1, keepdim=True) + 1e-6).sqrt()).bfloat16().reshape(2, R, HK * HD)
    v = torch.nn.functional.silu(r.normal(R, HV * HD)).bfloat16()
    decay = 1.0 + 15.0 * r.uniform(HV)                                    # exp(A_log)
    step = torch.exp(r.uniform(HV) * math.log(100.0) + math.log(1e-3))    # softplus(dt_bias), 0.001 .. 0.1
    bias = step + torch.log(-torch.expm1(-step))
    g = -decay * torch.nn.functional.softplus(r.normal(R, HV) + bias)
    s = {"c": c, "q": q.contiguous(), "k": k.contiguous(), "v": v, "g": g, "scale": HD ** -0.5,
         "beta": torch.sigmoid(r.normal(R, HV)).bfloat16() if c["delta"] else None}
    if c["op"] == "prompt":
        s["seq_ptr"] = _pointers(L)
        s["state"] = 0.1 * r.normal(S + 1, HV, HD, HD) if c["state"] else None
        # every other sequence goes on from a state of the pool, the first of them included; the others start anew
        s["src"] = torch.where(torch.arange(S, device="cuda") % 2 == 0, r.perm(S + 1)[:S].int(), -1).int() if c["state"] else None
        return s
    s["state"] = 0.1 * r.normal(S + 2, HV, HD, HD)
    s["slot"] = r.perm(S + 2)[:S].int()
    return s


# ---------------------------------------------------------------------------------------------------------- plain forms
def _write_plain(s):
    c, at = s["c"], s["slots"]
    page, off = at // c["page"], at % c["page"]
    for x, cache, scales in ((s["k"], s["kc"], s["ks"]), (s["v"], s["vc"], s["vs"])):
        x = x.transpose(0, 1)                     # [N, HKV, D]
        if scales is None:
            cache[page, :, off] = x
        else:
            stored, scale = _quantised(x)
            cache.view(torch.uint8)[page, :, off] = stored.view(torch.uint8)
            scales[page, :, off] = scale
    return [t for t in (s["kc"], s["vc"], s["ks"], s["vs"]) if t is not None]


def _gathered(cache, scales, page, off):
    """Rows of a cache as fp32 [tokens, HKV, D]."""
    if scales is None:
        return cache[page, :, off].float()
    return cache.view(torch.uint8)[page, :, off].view(torch.float8_e4m3fn).float() * scales[page, :, off][..., None]


def _read_plain(s):
    page, off = s["slots"] // s["c"]["page"], s["slots"] % s["c"]["page"]
    return [_gathered(x, sc, page, off).bfloat16().transpose(0, 1).contiguous()
            for x, sc in ((s["kc"], s["ks"]), (s["vc"], s["vs"]))]


def _tree_plain(s):
    c = s["c"]
    B, HKV, G, D, PS = c["B"], c["HKV"], c["G"], c["D"], c["page"]
    q_ptr, ctx = s["q_ptr"].long(), s["ctx"].long()
    N, most, width = s["q"].shape[1], c["n"], s["table"].shape[1] * PS
    dev = s["q"].device
    # rows and cache positions of the sequences, padded to the longest
    i, p = torch.arange(most, device=dev), torch.arange(width, device=dev)
    n = q_ptr[1:] - q_ptr[:-1]
    live = i[None] < n[:, None]                                                     # [B, most]
    row = torch.where(live, q_ptr[:-1, None] + i[None], 0)
    page = s["table"].long()[:, p // PS]
    here = (page >= 0) & (p[None] < (ctx + n)[:, None])
    k, v = (torch.where(here[..., None, None], _gathered(x, sc, page.clamp_min(0), p % PS), 0.0).transpose(1, 2)
            for x, sc in ((s["kc"], s["ks"]), (s["vc"], s["vs"])))                  # [B, HKV, width, D]
    q = s["q"].float()[:, row].reshape(HKV, G, B, most, D).permute(2, 0, 1, 3, 4).reshape(B, HKV, G * most, D)
    # what each row sees: the context, and of the drafted tokens what its bits (or the order) say
    j = (p[None] - ctx[:, None])[:, None].expand(B, most, width)
    if s["bits"] is None:
        drafted = j <= i[None, :, None]
    else:
        word = (j // 64).clamp(0, s["bits"].shape[1] - 1)
        drafted = (torch.gather(s["bits"][row], 2, word) >> (j % 64)) & 1 == 1
    sees = here[:, None] & live[..., None] & ((j < 0) | drafted)
    sees = sees[:, None, None].expand(B, 1, G, most, width).reshape(B, 1, G * most, width)
    score = (q @ k.transpose(-1, -2)) * s["scale"]
    score = torch.where(sees, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(top.isinf(), 0.0, top))
    total = weight.sum(-1, keepdim=True)
    out = torch.where(total > 0, (weight @ v) / total, 0.0)
    lse = torch.where(total > 0, top + torch.log(total), -math.inf)
    out = out.reshape(B, HKV * G, most, D).permute(0, 2, 1, 3)[live].reshape(N, HKV * G * D)
    return [out.bfloat16(), lse.reshape(B, HKV * G, most).permute(0, 2, 1)[live]]


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


def _prompt_plain(s):
    c, C = s["c"], CHUNK
    HK, G, S = c["HK"], c["G"], c["S"]
    HV, dev, ptr = HK * G, s["q"].device, s["seq_ptr"].long()
    R, chunks = s["q"].shape[0], max(1, -(-c["L"] // C))
    t = torch.arange(chunks * C, device=dev)
    live = t[None] < (ptr[1:] - ptr[:-1])[:, None]                                  # [S, chunks * C]
    row = torch.where(live, ptr[:-1, None] + t[None], 0)

    def laid(x, heads):   # [R, heads * w] -> fp32 [S, HV, chunks, C, w], zeros behind a sequence's end
        x = torch.where(live[..., None, None], x.float().reshape(R, heads, -1)[row], 0.0)
        x = x.reshape(S, chunks, C, heads, -1).permute(0, 3, 1, 2, 4)
        return x.repeat_interleave(HV // heads, 1)

    q, k, v = laid(s["q"], HK), laid(s["k"], HK), laid(s["v"], HV)
    sums = laid(s["g"], HV)[..., 0].double().cumsum(-1)                             # [S, HV, chunks, C]
    lower = torch.ones(C, C, device=dev).tril().bool()
    fade = torch.where(lower, sums[..., :, None] - sums[..., None, :], -math.inf).exp().float()
    from_start, to_end = sums.exp().float(), (sums[..., -1:] - sums).exp().float()
    within = fade * (q @ k.transpose(-1, -2))
    if c["delta"]:
        beta = laid(s["beta"], HV)
        inverse = _unit_lower_inverse(beta * (fade * (k @ k.transpose(-1, -2))).tril(-1))
    state = torch.zeros(S, HV, HD, HD, device=dev)
    if s["state"] is not None:
        src = s["src"].long()
        state = torch.where((src >= 0)[:, None, None, None], s["state"][src.clamp_min(0)], 0.0)
    out = torch.empty(S, HV, chunks, C, HD, device=dev)
    for m in range(chunks):
        u = v[:, :, m]
        if c["delta"]:
            u = inverse[:, :, m] @ (beta[:, :, m] * (u - from_start[:, :, m, :, None] * (k[:, :, m] @ state)))
        out[:, :, m] = from_start[:, :, m, :, None] * (q[:, :, m] @ state) + within[:, :, m] @ u
        state = from_start[:, :, m, -1, None, None] * state + (to_end[:, :, m, :, None] * k[:, :, m]).transpose(-1, -2) @ u
    o = (s["scale"] * out).permute(0, 2, 3, 1, 4).reshape(S, chunks * C, HV * HD)[live]
    return [o.bfloat16(), state]


def _step_plain(s):
    c, slot = s["c"], s["slot"].long()
    B, HK, HV = c["B"], c["HK"], c["HK"] * c["G"]
    q, k = (x.float().reshape(B, HK, HD).repeat_interleave(c["G"], 1) for x in (s["q"], s["k"]))
    u = s["v"].float().reshape(B, HV, HD)
    state = s["state"][slot] * s["g"].exp()[..., None, None]
    if c["delta"]:
        u = s["beta"].float()[..., None] * (u - (k[..., None, :] @ state)[..., 0, :])
    state = state + k[..., :, None] * u[..., None, :]
    s["state"][slot] = state
    o = s["scale"] * (q[..., None, :] @ state)[..., 0, :]
    return [o.reshape(B, HV * HD).bfloat16(), s["state"]]


# ------------------------------------------------------------------------------------------------------------- one pass
@functools.lru_cache(None)
def _package():
    from __graft_entry__ import load_package
    load_package()
    from open_jev_fast_amd import ext
    return ext


def run(s):
    op = s["c"]["op"]
    if own:
        ext = _package()
        if op == "write":
            ext.kv_cache_write(s["k"], s["v"], s["slots"], s["kc"], s["vc"], s["ks"], s["vs"])
            return [t for t in (s["kc"], s["vc"], s["ks"], s["vs"]) if t is not None]
        if op == "read":
            return list(ext.kv_cache_read(s["kc"], s["vc"], s["slots"], s["ks"], s["vs"]))
        if op == "tree":
            return list(ext.tree_attn(s["q"], s["kc"], s["vc"], s["table"], s["ctx"], s["q_ptr"], s["bits"], s["ks"],
                                      s["vs"], scale=s["scale"], want_lse=True))
        if op == "prompt":
            return list(ext.linattn_prompt(s["q"], s["k"], s["v"], s["g"], s["beta"], s["seq_ptr"], s["state"], s["src"],
                                           scale=s["scale"]))
        return [ext.linattn_step(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"], s["slot"], scale=s["scale"]),
                s["state"]]
    return {"write": _write_plain, "read": _read_plain, "tree": _tree_plain, "prompt": _prompt_plain,
            "step": _step_plain}[op](s)


# ------------------------------------------------------------------------------------------------- the same in 64 bits
def _e4m3_of(x):
    """x (64 bits, |x| <= 448) rounded to the nearest e4m3 value, ties to the even one."""
    size = x.abs().clamp_min(2.0 ** -6)
    unit = torch.exp2(torch.floor(torch.log2(size)) - 3)      # spacing: 3 bits behind the leading one, 2^-9 below 2^-6
    unit = torch.where(size / unit >= 16, unit * 2, torch.where(size / unit < 8, unit / 2, unit))
    return torch.round(x / unit) * unit                       # torch.round takes ties to even


def _exact_store(x):
    x = x.double()
    top = x.abs().amax(-1)
    e = torch.ceil(torch.log2(top / 448))
    e = torch.where(torch.exp2(e - 1) * 448 >= top, e - 1, torch.where(torch.exp2(e) * 448 < top, e + 1, e))
    scale = torch.where(top == 0, 1.0, torch.exp2(e.clamp_min(-126)))
    return _e4m3_of(x / scale[..., None]), scale


def _exact_cache(s):
    """Keys and values that the cache stands for, 64 bits [pages, HKV, page, D]."""
    return [x.double() if sc is None else x.float().double() * sc.double()[..., None]
            for x, sc in ((s["kc"], s["ks"]), (s["vc"], s["vs"]))]


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "write":
        page, off = s["slots"] // c["page"], s["slots"] % c["page"]
        stored, scales = [], []
        for x, cache, scale in ((s["k"], s["kc"], s["ks"]), (s["v"], s["vc"], s["vs"])):
            cache = cache.float().double()
            if scale is None:
                cache[page, :, off] = x.transpose(0, 1).double()
            else:
                scale = scale.double()
                cache[page, :, off], scale[page, :, off] = _exact_store(x.transpose(0, 1))
                scales.append(scale)
            stored.append(cache)
        return stored + scales
    if c["op"] == "read":
        flat = [x.transpose(1, 2).reshape(-1, c["HKV"], c["D"])[s["slots"]] for x in _exact_cache(s)]
        return [x.transpose(0, 1).contiguous() for x in flat]
    if c["op"] == "tree":
        return _exact_tree(s)
    return _exact_linear(s)


def _exact_tree(s):
    c = s["c"]
    HKV, G, D, PS = c["HKV"], c["G"], c["D"], c["page"]
    flat = [x.transpose(1, 2).reshape(-1, HKV, D) for x in _exact_cache(s)]
    n, ctx = _tree_lengths(c)
    outs, lses, at = [], [], 0
    for b in range(c["B"]):
        if n[b] == 0:
            continue
        pos = torch.arange(ctx[b] + n[b], device="cuda")
        slot = s["table"][b].long()[pos // PS] * PS + pos % PS
        k, v = (x[slot] for x in flat)                                    # [positions, HKV, D]
        q = s["q"][:, at:at + n[b]].double()                              # [HQ, n, D]
        sees = torch.ones(n[b], ctx[b] + n[b], dtype=torch.bool, device="cuda")
        if s["bits"] is None:
            sees[:, ctx[b]:] = torch.arange(n[b], device="cuda")[:, None] >= torch.arange(n[b], device="cuda")
        else:
            words = s["bits"][at:at + n[b]]
            shift = torch.arange(64, device="cuda")
            each = ((words[..., None] >> shift) & 1).bool().reshape(n[b], -1)
            sees[:, ctx[b]:] = each[:, :n[b]]
        out, lse = [], []
        for h in range(HKV * G):
            score = (q[h] @ k[:, h // G].T) * s["scale"]
            score = score.masked_fill(~sees, -math.inf)
            norm = torch.logsumexp(score, -1)
            out.append(torch.exp(score - norm[:, None]) @ v[:, h // G])
            lse.append(norm)
        outs.append(torch.stack(out, 1).reshape(n[b], -1))
        lses.append(torch.stack(lse, 1))
        at += n[b]
    return [torch.cat(outs), torch.cat(lses)]


def _exact_linear(s):
    """Token by token."""
    c = s["c"]
    G, HK = c["G"], c["HK"]
    HV = HK * G
    if c["op"] == "step":
        L, held = [1] * c["B"], s["state"].double()
        state = held[s["slot"].long()]
    else:
        L = _prompt_lengths(c)
        state = torch.zeros(c["S"], HV, HD, HD, dtype=torch.float64, device="cuda")
        if s["state"] is not None:
            for i, at in enumerate(s["src"].tolist()):
                if at >= 0:
                    state[i] = s["state"][at].double()
    first = s["seq_ptr"][:-1].long() if c["op"] == "prompt" else torch.arange(c["B"], device="cuda")
    length = torch.tensor(L, device="cuda")
    R = s["q"].shape[0]
    q, k = (x.double().reshape(R, HK, HD) for x in (s["q"], s["k"]))
    v, g = s["v"].double().reshape(R, HV, HD), s["g"].double().exp()
    beta = s["beta"].double() if c["delta"] else None
    out = torch.zeros(R, HV, HD, dtype=torch.float64, device="cuda")
    for t in range(max(L)):
        on = (length > t).nonzero()[:, 0] if min(L) <= t else None        # all of them while the shortest lasts
        row = first + t if on is None else first[on] + t
        one = state if on is None else state[on]
        kt = k[row].repeat_interleave(G, 1)
        one = one * g[row][..., None, None]
        u = v[row]
        if c["delta"]:
            u = beta[row][..., None] * (u - torch.matmul(kt[..., None, :], one)[..., 0, :])
        one = one + kt[..., None] * u[..., None, :]
        out[row] = s["scale"] * torch.matmul(q[row].repeat_interleave(G, 1)[..., None, :], one)[..., 0, :]
        if on is None:
            state = one
        else:
            state[on] = one
    out = out.reshape(R, HV * HD)
    if c["op"] == "step":
        held[s["slot"].long()] = state
        return [out, held]
    return [out, state]
