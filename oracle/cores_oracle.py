"""CPU oracle of the attention cores and the paged cache, in 64 bits — TEST INFRASTRUCTURE ONLY.

Written from the definitions, one row or token at a time, apart from any kernel: only tests may import it.

  cache_store    a row x of D values -> (e4m3 bytes, scale): scale the smallest power of two 2^e, e >= -126, with
                 max |x| <= 448 scale over the finite values (1 for zeros); x / scale to the nearest of the 256 e4m3 values,
                 ties to the even code; NaN for a value that is not finite
  cache_values   what a cache stands for, fp64
  tree_attn      attention of drafted tokens over a paged cache, with a bound of the kernel's error beside it
  linattn        linear attention token by token, with a bound of the kernel's error beside it

The bounds follow the roundings a kernel is entitled to: half a step of bf16, u = 2^-8, on its output and on the weights
that a matrix product takes in bf16; fp32 sums; and, for linear attention, factors of two or three bf16 pieces (u^2 = 2^-16
and u^3 = 2^-24 together).
"""
import math

import torch

U = 2.0 ** -8     # half a step of bf16, relative
F = 2.0 ** -24    # half a step of fp32


def e4m3_table():
    """The value of every e4m3 code (OCP, no infinities; 0x7f and 0xff are NaN), fp64 [256]."""
    vals = []
    for code in range(256):
        e, m = code >> 3 & 15, code & 7
        x = math.nan if e == 15 and m == 7 else (m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
        vals.append(-x if code & 128 else x)
    return torch.tensor(vals, dtype=torch.float64)


_TABLE = e4m3_table()


def cache_store(x):
    """x bf16 [.., D] -> (values fp64 [.., D] that the bytes stand for before the scale, scale fp64 [..])."""
    x = x.double()
    fine = torch.isfinite(x)
    top = torch.where(fine, x.abs(), 0.0).amax(-1)
    scale = torch.ones_like(top)
    for at in (top > 0).nonzero():
        at = tuple(at.tolist())
        e = -126
        while 448.0 * 2.0 ** e < top[at].item():
            e += 1
        scale[at] = 2.0 ** e
    pos = _TABLE[:127]                                     # codes 0 .. 126 ascend
    y = torch.where(fine, x, 0.0) / scale[..., None]
    hi = torch.searchsorted(pos, y.abs().contiguous()).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    dl, dh = y.abs() - pos[lo], pos[hi] - y.abs()
    code = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    v = torch.copysign(pos[code], y)
    return torch.where(fine, v, math.nan), scale


def cache_values(c, s):
    """fp64 values of a cache [pages, HKV, page, D] (bf16, or float8_e4m3fn with its scales)."""
    if s is None:
        return c.double()
    return _TABLE[c.view(torch.uint8).long()] * s.double()[..., None]


def tree_attn(q, kc, vc, ks, vs, table, ctx, q_ptr, bits, scale):
    """(out fp64 [N, HQ, D], lse fp64 [N, HQ], bound of |out - kernel|, bound of |lse - kernel|)."""
    HQ, N, D = q.shape
    pages, HKV, page, _ = kc.shape
    K, V = cache_values(kc, ks), cache_values(vc, vs)
    out, lse = torch.zeros(N, HQ, D, dtype=torch.float64), torch.full((N, HQ), -math.inf, dtype=torch.float64)
    bo, bl = torch.zeros_like(out), torch.zeros_like(lse)
    for b in range(ctx.numel()):
        first, end = int(q_ptr[b]), int(q_ptr[b + 1])
        c = max(0, int(ctx[b]))
        for n in range(first, end):
            rows = []
            for p in range(min(c + end - first, table.shape[1] * page)):
                j = p - c
                if j >= 0:
                    if bits is None:
                        see = j <= n - first
                    else:
                        see = j < 64 * bits.shape[1] and (int(bits[n, j // 64]) >> (j % 64)) & 1
                    if not see:
                        continue
                t = int(table[b, p // page])
                if 0 <= t < pages:
                    rows.append((t, p % page))
            if not rows:
                continue
            t, o = torch.tensor([r[0] for r in rows]), torch.tensor([r[1] for r in rows])
            for h in range(HQ):
                k, v = K[t, h // (HQ // HKV), o], V[t, h // (HQ // HKV), o]
                x = q[h, n].double()
                s = (k @ x) * scale
                lse[n, h] = torch.logsumexp(s, 0)
                w = torch.softmax(s, 0)
                out[n, h] = w @ v
                # a score: D products summed in fp32, scaled, taken to base two, less the maximum, its exponential
                es = ((k.abs() @ x.abs()) * abs(scale) * (D + 8) * F + (s.abs() + s.abs().max() + 8) * 4 * F).max().item()
                sums = len(rows) * F
                # every weight off by 2 es + sums and rounded to bf16, the result rounded to bf16; the smallest bf16 step
                bo[n, h] = (w @ v.abs()) * (U + 2 * es + 2 * sums + 4 * F) * 1.01 + U * out[n, h].abs() * 1.01 + 1e-38
                bl[n, h] = es + sums + 4 * F * (1 + lse[n, h].abs())
    return out, lse, bo, bl


def linattn(q, k, v, g, beta, lengths, state, scale):
    """Sequences one after the other in the rows, state fp64 [S, HV, 128, 128] or None. (o fp64 [R, HV, 128], states,
    bound of |o - kernel| [R, HV, 128], bound of the states' error in the 2-norm of each head [S, HV]).

    A kernel with two bf16 pieces or more in the state's products commits at each token errors of at most e = 2 u^2 times
    what it adds up: S^T k, the u of the tokens before in its chunk of 64, and the new state. An error in S is carried on
    by e^g (I - beta k k^T), which is no larger than e^g while beta |k|^2 <= 2: the bound E of the state's error follows
    the recurrence E <- e^g E + committed, and |o| is off by scale |q| E, by u on each factor that it takes in bf16 and
    by its own rounding."""
    R, HV = g.shape
    HK = k.shape[1] // 128
    G = HV // HK
    q, k, v = (x.double().reshape(R, -1, 128) for x in (q, k, v))
    q, k = q.repeat_interleave(G, 1), k.repeat_interleave(G, 1)
    g = g.double()
    beta = None if beta is None else beta.double()
    S = len(lengths)
    st = torch.zeros(S, HV, 128, 128, dtype=torch.float64) if state is None else state.double().clone()
    o, bo = torch.zeros(R, HV, 128, dtype=torch.float64), torch.zeros(R, HV, 128, dtype=torch.float64)
    E = torch.zeros(S, HV, dtype=torch.float64)
    e = 2 * U * U
    at = 0
    for s in range(S):
        M, err = st[s], torch.zeros(HV, dtype=torch.float64)
        us = []
        for t in range(lengths[s]):
            r = at + t
            a = g[r].exp()
            M = M * a[:, None, None]
            u = v[r]
            if beta is not None:
                u = beta[r][:, None] * (u - (M * k[r][..., None]).sum(1))
            us = (us if t % 64 else []) + [u]
            before = torch.stack(us).norm(dim=-1).sum(0)
            kn = k[r].norm(dim=-1)
            held = M.norm(dim=(1, 2))
            M = M + k[r][..., None] * u[:, None, :]
            err = a * err + e * (kn * (held * kn + before * (1 + kn) + v[r].norm(dim=-1)) + M.norm(dim=(1, 2)))
            o[r] = scale * (M * q[r][..., None]).sum(1)
            inside = sum(x.abs() for x in us) * kn[:, None]       # the chunk's tokens, weights and values in bf16
            col = M.norm(dim=1) + inside + (held + before * kn)[:, None] * U
            qn = q[r].norm(dim=-1)[:, None]
            bo[r] = abs(scale) * (qn * err[:, None] + 2.1 * U * qn * col) + 1.01 * U * o[r].abs() + 1e-38
        st[s], E[s] = M, err
        at += lengths[s]
    return o, st, bo, E


def linattn_chunk(q, k, v, g, beta, lengths, state, scale):
    """linattn for sequences of at most 64 tokens from given states, with bounds entry by entry instead of by norms:
    (o fp64 [R, HV, 128], states, bound of |o - kernel| [R, HV, 128], bound of |states - kernel| [S, HV, 128, 128]).

    They hold for a kernel that takes the tokens of a sequence at once,
      A_ij = beta_i e^(G_i - G_j) k_i . k_j (j < i),  P_ij = e^(G_i - G_j) q_i . k_j (j <= i),  T = (I + A)^-1 diag(beta),
      X = V - diag(e^G) K S0,  U = T X,  O = scale (diag(e^G) Q S0 + P U),  S = e^(G_n) S0 + K^T diag(e^(G_n - G)) U
    (T the identity and U = V without beta), sums in fp32, and lets S0, X, diag(e^(G_n - G)) T and U into the products that
    make states as three bf16 pieces, S0, P T and X into those that make outputs as two. Of x, hi = bf16(x) and lo =
    bf16(x - hi) leave out at most U^2 |x|, a third piece U^3 |x|; a product of two such factors leaves out its smallest, lo
    lo or three of U^3, besides. A sum of n terms is off by at most 2 F n times the sum of their magnitudes, in any order and
    also where additions are cut off instead of rounded; n grows with the pieces. An exponential is off by its argument's
    rounding and a step of its own. The errors go through the formulas in magnitudes."""
    R, HV = g.shape
    HK = k.shape[1] // 128
    G = HV // HK
    q, k, v = (x.double().reshape(R, -1, 128) for x in (q, k, v))
    q, k = q.repeat_interleave(G, 1), k.repeat_interleave(G, 1)
    g, beta = g.double(), None if beta is None else beta.double()
    S = len(lengths)
    st, o = torch.zeros(S, HV, 128, 128, dtype=torch.float64), torch.zeros(R, HV, 128, dtype=torch.float64)
    bs, bo = torch.zeros_like(st), torch.zeros_like(o)
    two, three, dot = U * U, U ** 3, 2 * F * 256
    tiny = 1e-35                                                # factors below the smallest fp32 step

    def expo(x):
        """e^x and its relative error: the argument, to base two, in fp32, and a step of fp32 for the exponential."""
        return x.exp(), 1.01 * F * x.abs() + 3 * F

    at = 0
    for s, n in enumerate(lengths):
        assert n <= 64
        for h in range(HV):
            S0 = torch.zeros(128, 128, dtype=torch.float64) if state is None else state[s, h].double()
            if n == 0:
                st[s, h] = S0
                continue
            r = slice(at, at + n)
            Q, K, V = q[r, h], k[r, h], v[r, h]
            cum = g[r, h].cumsum(0)
            low = torch.ones(n, n, dtype=torch.float64).tril()
            fade, dfade = expo(torch.where(low > 0, cum[:, None] - cum[None], 0.0))
            fade = fade * low
            since, dsince = (x[:, None] for x in expo(cum))
            to, dto = (x[:, None] for x in expo(cum[-1] - cum))
            KS, QS, SA = K @ S0, Q @ S0, S0.abs()
            dKS, dQS = ((left + 2 * dot) * (x.abs() @ SA) for x, left in ((K, three), (Q, two)))
            P = fade * (Q @ K.T)
            dP = fade * (dot * (Q.abs() @ K.abs().T) + (dfade + 2 * F) * (Q @ K.T).abs())
            if beta is None:
                X, dX, T, dT = V, torch.zeros_like(V), None, None
                W, dW = P, dP                                       # what X meets for the outputs
                u, du = V, torch.zeros_like(V)
                end, dend = to * V, (dto + F) * (to * V).abs()      # U, decayed to the end
            else:
                b = beta[r, h][:, None]
                A = (b * fade * (K @ K.T)).tril(-1)
                dA = (b.abs() * fade * (dot * (K.abs() @ K.abs().T) + (dfade + 3 * F) * (K @ K.T).abs())).tril(-1)
                I = torch.eye(n, dtype=torch.float64)
                inv = torch.linalg.solve_triangular(I + A, I, upper=False)
                # forward substitution is off by |T| |L| |T| F n; put together from blocks of 16, each block row passes on
                # what the ones above are off by, through |T| |L| again
                E, own = inv.abs() @ (I + A).abs(), torch.zeros_like(A)
                power = 2 * F * (n + 2) * inv.abs()
                for _ in range(1 if n <= 16 else 4):
                    power = E @ power
                    own = own + power
                T = inv * b.T
                dT = (inv.abs() @ dA @ inv.abs() + own) * b.abs().T + F * T.abs()
                X = V - since * KS
                dX = since * dKS + (dsince + 2 * F) * (since * KS).abs() + F * X.abs()
                W = P @ T
                dW = P.abs() @ dT + dP @ T.abs() + 2 * F * n * (P.abs() @ T.abs())
                W, dW = W.tril(), dW.tril()
                u = T @ X
                both = (6 * three + 2 * F * 6 * n) * (T.abs() @ X.abs())
                end, dend = to * u, to * (T.abs() @ dX + dT @ X.abs() + both + (dto + 2 * F) * (T.abs() @ X.abs()))
            S1, all_, dall = to * u, since[-1], dsince[-1]
            st[s, h] = all_ * S0 + K.T @ S1
            bs[s, h] = ((dall + 4 * F) * all_ * SA + K.abs().T @ (dend + three * end.abs())
                        + 2 * F * (3 * n + 2) * (K.abs().T @ end.abs())) * 1.01 + tiny
            o[r, h] = scale * (since * QS + P @ u)
            left = (3 if beta is not None else 1) * two
            err = since * dQS + (dsince + 3 * F) * (since * QS).abs() + W.abs() @ dX + dW @ X.abs()
            err = err + (left + 2 * F * (3 * n + 4)) * (W.abs() @ X.abs()) + 2 * F * (since * QS).abs()
            bo[r, h] = (abs(scale) * err * (1 + U) + U * o[r, h].abs()) * 1.01 + tiny
        at += n
    return o, st, bo, bs
