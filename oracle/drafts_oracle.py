"""CPU oracle of the operators around drafted tokens, in 64 bits — TEST INFRASTRUCTURE ONLY.

Written from the definitions, one row, token or page at a time, apart from any kernel: only tests may import it.

  verify        drafted tokens against the target's distributions, each rejection's distribution made from the one before it
  linattn_tree  linear attention of a tree of tokens by a state for every row, with a bound of the kernel's error beside it
  linattn_keep  a state token by token, with a bound of the kernel's error beside it
  keep_rows     kept rows of a paged cache, moved
  resize, fork  tables, counts and contexts of a paged cache
"""
import math

import torch

U = 2.0 ** -8     # half a step of bf16, relative
F = 2.0 ** -24    # half a step of fp32


def spans(q_ptr, N):
    """(first row, rows) of each sequence: pointers clamped to [0, N], none below the ones before it."""
    at, out = 0, []
    p = [min(max(int(x), 0), N) for x in q_ptr]
    for b in range(len(p) - 1):
        at = max(at, p[b])
        end = max(at, p[b + 1])
        out.append((at, end - at))
    return out


def target(x, t):
    """The distribution of a row of logits at temperature t, or None."""
    x = x.double()
    if bool(torch.isnan(x).any()) or bool((x == math.inf).any()) or bool((x == -math.inf).all()):
        return None
    if not t > 0:
        p = torch.zeros_like(x)
        p[int((x == x.max()).nonzero()[0, 0])] = 1.0
        return p
    top = x.max()
    e = torch.where(x == -math.inf, 0.0, torch.exp((x - top) / t))
    return e / e.sum()


def verify(logits, tokens, q_ptr, u, parents, probs, temperature):
    """(path [N], count [B], next [B], the least relative distance of a test or draw from its border)."""
    N, V = logits.shape
    B = len(q_ptr) - 1
    path, count, nxt, near = [-1] * N, [0] * B, [-1] * B, math.inf
    for b, (first, n) in enumerate(spans(q_ptr, N)):
        if n == 0:
            continue
        t = 1.0 if temperature is None else float(temperature[b])
        t = t if t > 0 else 0.0
        cur, taken = 0, [0]
        while True:
            own = target(logits[first + cur], t)
            nxt_row = None
            if own is not None:
                p, left = own, True
                for j in range(cur + 1, n):
                    above = j - 1 if parents is None else int(parents[first + j])
                    if above != cur:
                        continue
                    x = int(tokens[first + j])
                    q = None
                    if probs is not None and t > 0:
                        q = probs[first + cur].double()
                        q = torch.where(q > 0, q, 0.0)
                    px = float(p[x]) if 0 <= x < V and left else 0.0
                    qx = (1.0 if q is None else float(q[x])) if 0 <= x < V else (1.0 if q is None else 0.0)
                    test = float(u[first + j]) * qx
                    if test > 0 and px > 0 and t > 0:
                        near = min(near, abs(test / px - 1))
                    if test < px:
                        nxt_row = j
                        break
                    if t > 0:
                        rest = p.clone()
                        if q is None:
                            if 0 <= x < V:
                                rest[x] = 0.0
                        else:
                            rest = torch.where(q > 0, (p - q).clamp_min(0), p)
                        total = float(rest.sum())
                        left = left and total > 0
                        p = rest / total if total > 0 else torch.zeros_like(p)
            if nxt_row is None:
                break
            cur = nxt_row
            taken.append(cur)
        path[first:first + len(taken)] = taken
        count[b] = len(taken)
        if own is None:
            continue
        if not left:
            p = own
        sums = p.cumsum(0)
        level = (float(u[first]) if t > 0 else 0.0) * float(sums[-1])
        over = ((sums > level) & (p > 0)).nonzero()
        nxt[b] = int(over[0, 0]) if len(over) else int((p > 0).nonzero()[-1, 0])
        if t > 0 and level > 0:
            near = min(near, float((sums / level - 1).abs().min()))
    return path, count, nxt, near


# ----------------------------------------------------------------------------------------------------- linear attention
def _heads(x, HV):
    R = x.shape[0]
    x = x.double().reshape(R, -1, 128)
    return x.repeat_interleave(HV // x.shape[1], 1)


def above(parents, first, j):
    p = j - 1 if parents is None else int(parents[first + j])
    return p if 0 <= p < j else -1


def linattn_tree(q, k, v, g, beta, state, slot, q_ptr, parents, scale):
    """(o fp64 [N, HV, 128], bound of |o - kernel|). Rows of no sequence and of a negative slot are 0, those of a slot that is
    not there NaN.

    The bounds hold for a kernel that takes a sequence's rows at once,
      A_ij = beta_i e^(G_i - G_j) k_i . k_j, P_ij = e^(G_i - G_j) q_i . k_j, T = (I + A)^-1 diag(beta),
      X = V - diag(e^G) K S0,  U = T X,  O = scale (diag(e^G) Q S0 + P U)
    with j an ancestor of i (in P also i itself), sums in fp32, S0, X, U and the matrices as two bf16 pieces or better: of a
    factor hi + lo leaves out U^2, a product of two such a third U^2. A sum of n terms is off by 2 F n of their magnitudes. The
    errors go through the formulas in magnitudes."""
    N, HV = g.shape
    q, k, v = _heads(q, HV), _heads(k, HV), v.double().reshape(N, HV, 128)
    g, beta = g.double(), None if beta is None else beta.double()
    o, bo = torch.zeros(N, HV, 128, dtype=torch.float64), torch.zeros(N, HV, 128, dtype=torch.float64)
    two, dot, tiny = U * U, 2 * F * 256, 1e-35
    for b, (first, n) in enumerate(spans(q_ptr, N)):
        s = int(slot[b])
        if n == 0 or s < 0:
            continue
        if s >= state.shape[0]:
            o[first:first + n] = math.nan
            continue
        up = [above(parents, first, j) for j in range(n)]
        seen = torch.eye(n, dtype=torch.float64)
        for j in range(n):
            if up[j] >= 0:
                seen[j] = torch.maximum(seen[j], seen[up[j]])
        r = slice(first, first + n)
        for h in range(HV):
            S0 = state[s, h].double()
            # the values: a state for every row
            states = []
            for j in range(n):
                M = (S0 if up[j] < 0 else states[up[j]]) * g[first + j, h].exp()
                x = v[first + j, h]
                if beta is not None:
                    x = beta[first + j, h] * (x - M.T @ k[first + j, h])
                states.append(M + k[first + j, h][:, None] * x[None])
                o[first + j, h] = scale * (states[j].T @ q[first + j, h])
            # the bounds
            Q, K, V = q[r, h], k[r, h], v[r, h]
            gc = g[r, h].clamp_min(-200.0)
            G = seen @ gc
            fade = torch.where(seen > 0, (G[:, None] - G[None]).exp(), 0.0)
            dfade = 1.01 * F * torch.where(seen > 0, (G[:, None] - G[None]).abs(), 0.0) + 3 * F
            since, dsince = G.exp()[:, None], (1.01 * F * G.abs() + 3 * F)[:, None]
            steps = seen.sum(-1)[:, None] * 4 * F                  # a decay made as a product over the path
            dsince, dfade = dsince + steps, dfade + steps
            KS, QS, SA = K @ S0, Q @ S0, S0.abs()
            dKS, dQS = ((two + 2 * dot) * (x.abs() @ SA) for x in (K, Q))
            P = fade * (Q @ K.T)
            dP = fade * (dot * (Q.abs() @ K.abs().T) + (dfade + 2 * F) * (Q @ K.T).abs())
            if beta is None:
                u, du = V, torch.zeros_like(V)
            else:
                c = beta[r, h][:, None]
                low = seen - torch.eye(n, dtype=torch.float64)
                A = c * fade * low * (K @ K.T)
                dA = c.abs() * fade * low * (dot * (K.abs() @ K.abs().T) + (dfade + 3 * F) * (K @ K.T).abs())
                I = torch.eye(n, dtype=torch.float64)
                inv = torch.linalg.solve_triangular(I + A, I, upper=False)
                E, own = inv.abs() @ (I + A).abs(), torch.zeros_like(A)
                power = 2 * F * (n + 2) * inv.abs()
                for _ in range(-(-n // 16)):
                    power = E @ power
                    own = own + power
                T = inv * c.T
                dT = (inv.abs() @ dA @ inv.abs() + own) * c.abs().T + F * T.abs()
                X = V - since * KS
                dX = since * dKS + (dsince + 2 * F) * (since * KS).abs() + F * X.abs()
                u = T @ X
                du = T.abs() @ dX + dT @ X.abs() + (3 * two + 2 * F * 3 * n) * (T.abs() @ X.abs())
            err = since * dQS + (dsince + 3 * F) * (since * QS).abs() + P.abs() @ du + dP @ u.abs()
            err = err + (3 * two + 2 * F * (3 * n + 4)) * (P.abs() @ u.abs()) + 2 * F * (since * QS).abs()
            bo[r, h] = (abs(scale) * err * (1 + U) + U * o[r, h].abs()) * 1.01 + tiny
    return o, bo


def linattn_keep(k, v, g, beta, state, slot, q_ptr, path, count):
    """(states fp64, bound of |states - kernel|), the recurrence in fp32, entry by entry."""
    N, HV = g.shape
    k, v = _heads(k, HV), v.double().reshape(N, HV, 128)
    st, bs, named = state.double().clone(), torch.zeros(state.shape, dtype=torch.float64), set()
    for b, (first, n) in enumerate(spans(q_ptr, N)):
        s = int(slot[b])
        if s in named or not 0 <= s < state.shape[0]:
            continue
        named.add(s)
        for i in range(min(n, int(count[b]))):
            r = int(path[first + i])
            if not 0 <= r < n:
                continue
            r += first
            a = g[r].double().exp()[:, None, None]
            K, x = k[r], v[r]
            M, dM = a * st[s], a * bs[s]
            dM = dM + (1.01 * F * g[r].double().abs().clamp_max(200.0)[:, None, None] + 4 * F) * M.abs()
            dx = torch.zeros_like(x)
            if beta is not None:
                c = beta[r].double()[:, None]
                y = (M * K[..., None]).sum(1)
                dy = (dM * K.abs()[..., None]).sum(1) + 2 * F * 128 * (M.abs() * K.abs()[..., None]).sum(1)
                dx = c.abs() * (dy + 2 * F * (x - y).abs())
                x = c * (x - y)
                dx = dx + F * x.abs()
            st[s] = M + K[..., None] * x[:, None, :]
            bs[s] = dM + K.abs()[..., None] * (dx + 2 * F * x.abs())[:, None, :] + F * st[s].abs()
        bs[s] = bs[s] * 1.01 + 1e-35
    return st, bs


# ---------------------------------------------------------------------------------------------------------------- cache
def keep_rows(caches, table, ctx, q_ptr, path, count, page):
    """caches: tensors [layers, pages, HKV, page, ..], changed in place."""
    N, pages = len(path), caches[0].shape[1]
    before = [c.clone() for c in caches]
    for b, (first, n) in enumerate(spans(q_ptr, N)):
        c = max(0, int(ctx[b]))

        def place(pos):
            if pos // page >= table.shape[1]:
                return None
            t = int(table[b, pos // page])
            return (t, pos % page) if 0 <= t < pages else None

        for i in range(min(n, int(count[b]))):
            r = int(path[first + i])
            if r <= i or r >= n:
                continue
            src, dst = place(c + r), place(c + i)
            if src is None or dst is None:
                continue
            for x, y in zip(caches, before):
                x[:, dst[0], :, dst[1]] = y[:, src[0], :, src[1]]


def _take(refs):
    for t in range(len(refs)):
        if refs[t] <= 0:
            refs[t] = 1
            return t
    return -1


def resize(table, refs, tokens, page):
    """Lists, changed in place; missing."""
    pages, MP = len(refs), len(table[0]) if table else 0
    for b, row in enumerate(table):
        if tokens[b] < 0:
            continue
        for i in range(-(-tokens[b] // page), MP):
            if 0 <= row[i] < pages:
                refs[row[i]] -= 1
            row[i] = -1
    missing = []
    for b, row in enumerate(table):
        miss = 0
        if tokens[b] >= 0:
            want = -(-tokens[b] // page)
            for i in range(min(want, MP)):
                if not 0 <= row[i] < pages:
                    row[i] = _take(refs)
                    miss += row[i] < 0
            miss += max(0, want - MP)
        missing.append(miss)
    return missing


def fork(table, ctx, refs, src, page):
    """Lists, changed in place; pairs."""
    pages, B, MP = len(refs), len(table), len(table[0]) if table else 0
    old, length = [list(r) for r in table], list(ctx)
    pairs, held = [(-1, -1)] * B, []
    ok = lambda t: 0 <= t < pages  # noqa: E731
    for b in range(B):
        if src[b] != b:
            for t in old[b]:
                if ok(t):
                    refs[t] -= 1
    for b in range(B):
        s = src[b]
        if s == b:
            continue
        n = max(0, length[s]) if 0 <= s < B else 0
        full = min(n // page, MP)
        table[b] = [old[s][i] if 0 <= s < B and i < full and ok(old[s][i]) else -1 for i in range(MP)]
        for t in table[b]:
            if t >= 0:
                refs[t] += 1
        ctx[b] = n
        if n > full * page and full < MP and ok(old[s][full]):
            pairs[b] = (old[s][full], -1)
            refs[old[s][full]] += 1
            held.append(old[s][full])
    for b in range(B):
        if pairs[b][0] >= 0:
            t = _take(refs)
            pairs[b] = (pairs[b][0], t)
            full = min(ctx[b] // page, MP)
            if t >= 0:
                table[b][full] = t
            else:
                ctx[b] = full * page
    for t in held:
        refs[t] -= 1
    return pairs
