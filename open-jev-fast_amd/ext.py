"""Projection-path functions of the reference's kernel extension `K` (src/ext.py:6-29), on libojx.

Same names, arguments, return values and error behaviour (RuntimeError) as the reference's torch-extension
functions, for the entry points on the projection path:

    add_rmsnorm(x, delta, w1, rowmask, eps) -> [h, hn]        src/kernels.cu:41-73, 755-767
    add_rmsnorm_sk(x, parts, w1, rowmask, eps) -> [h, hn]     src/kernels.cu:475-515, 886-900
    add_rmsnorm_sk2(x, parts, w1, rowmask, eps) -> [h, hn]    src/kernels.cu:1444-1501 (S in 2..4)
    silu_mul(gu) -> out                                       src/kernels.cu:76-89, 769-777
    silu_mul_lut(gu, tab) -> out                              src/kernels.cu:1304-1331
    act_tables(like) -> [silu_b, sig_f]                       src/kernels.cu:1288-1301
    head_scores(hn, lastidx, w, bias) -> scores              src/server.py:37 (mdl.head(hn[lastidx].float()))

plus the fused projections that replace GEMM + epilogue pairs (mm, mm_silu_mul, mm_residual_rmsnorm,
mm_splitk_f32) and pack_gate_up, the weight layout of the fused gate-up.

Tensors must be contiguous GPU tensors (the reference's CHECK, src/kernels.cu:10); outputs come from torch's
allocator on their inputs' device and every launch goes on torch's current stream, so all of it can be captured in a
CUDA/HIP graph.
"""
import ctypes
import functools
import weakref

import torch

from . import _lib
from ._lib import KIND_PLAIN, KIND_RESIDUAL, KIND_SILU_MUL, check, lib


# The current stream of the current device, as the integer handle the C-ABI takes. torch.cuda.current_stream() builds a
# Stream object around the same two lookups (measured 1.6 us a call on the host, 0.2 without), and each entry point asks
# once per call. (A build of torch without GPU support has neither; nothing here runs there.)
_current_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream():
    return _current_raw_stream(torch._C._cuda_getDevice())


def _ptr(t):
    """A tensor's address for a c_void_p argument (ctypes converts the integer itself)."""
    return t.data_ptr() if t is not None else None


def _chk(t, name, dtype=None):
    if t is None:
        raise RuntimeError(f"{name} must be a tensor")
    if not (t.is_cuda and t.is_contiguous()):
        raise RuntimeError(f"{name} must be contiguous CUDA")
    if dtype is not None and t.dtype is not dtype:
        raise RuntimeError(f"{name} must be {dtype}, got {t.dtype}")


def _cfgp(cfg):
    if cfg is None:
        return None
    if not isinstance(cfg, _lib.OjxCfg):
        cfg = _lib.OjxCfg(*cfg)
    return ctypes.byref(cfg)


_WS = {}        # (device index, stream handle) -> the workspace handed to that stream's eager calls and captures
_WS_KEEP = []   # every workspace a graph capture has used: kept alive for the life of the process


def _workspace(M, N, K, kind, cfg, device):
    """Workspace of one call: split-K fp32 planes or stream-K partial tiles (scratch, contents irrelevant on entry).

    One buffer per stream of each device is kept and grown as needed, so calls on different streams may overlap (the
    library gives each stream its own set of arrival counters for the one-launch plans too). A graph capture records the buffer's address, so a buffer
    that a capture has used is not freed while graphs may replay: when a later call needs a larger one, the old
    buffer moves to _WS_KEEP instead of going back to the caching allocator (where a replay would write into memory
    that other tensors may own by then). The larger buffer becomes the device's buffer for every later call,
    eager or captured, so the kept memory grows only with the largest workspace seen per stream, not with the number
    of captures. release_workspaces() drops the kept buffers once the caller's graphs are gone. A captured graph
    replayed on another stream keeps the capture stream's workspace: replays that overlap with calls on the capture
    stream race on it."""
    n = lib().ojx_workspace_bytes(M, N, K, kind, _cfgp(cfg))
    if n < 0:
        check(1)
    if n == 0:
        return None, 0
    key = (device.index, _current_raw_stream(device.index))  # a GPU tensor's device: the index is set
    ws = _WS.get(key)
    capturing = torch._C._cuda_isCurrentStreamCapturing()
    if ws is not None and ws[0].numel() >= n:
        if capturing and not ws[1]:
            _WS[key] = ws = (ws[0], True)
            _WS_KEEP.append(ws[0])
        return ws[0], ws[0].numel()
    buf = torch.empty(max(n, 1 << 20), dtype=torch.uint8, device=device)
    _WS[key] = (buf, capturing)   # the old buffer, if a capture used it, stays alive in _WS_KEEP
    if capturing:
        _WS_KEEP.append(buf)
    return buf, buf.numel()


def release_workspaces():
    """Frees the workspace buffers kept for captured graphs (and the current ones). Call it only after every graph
    captured with this module's calls has been destroyed: a later replay of such a graph would write into freed
    memory."""
    _WS.clear()
    _WS_KEEP.clear()


def _chk_norm(w1, rowmask, M, H):
    """RMSNorm operands: w1 fp32 [H]; rowmask (optional) int32 [M]. The kernels read exactly that many."""
    _chk(w1, "w1", torch.float32)
    if w1.numel() != H:
        raise RuntimeError(f"w1 must have H={H} elements, got {w1.numel()}")
    if rowmask is not None:
        _chk(rowmask, "rowmask", torch.int32)
        if rowmask.numel() != M:
            raise RuntimeError(f"rowmask must have M={M} elements, got {rowmask.numel()}")


# ------------------------------------------------------------------------------------------------ epilogues
def add_rmsnorm(x, delta, w1, rowmask, eps):
    _chk(x, "x", torch.bfloat16)
    M, H = x.shape
    _chk_norm(w1, rowmask, M, H)
    hn = torch.empty_like(x)
    if delta is not None:
        _chk(delta, "delta", torch.bfloat16)
        if tuple(delta.shape) != (M, H):
            raise RuntimeError(f"delta {tuple(delta.shape)} must match x {tuple(x.shape)}")
        h = torch.empty_like(x)
    else:
        h = x
    check(lib().ojx_add_rmsnorm(_ptr(x), _ptr(delta), _ptr(w1), _ptr(rowmask), float(eps),
                                _ptr(h) if delta is not None else None, _ptr(hn), M, H, _stream()))
    return [h, hn]


def add_rmsnorm_sk(x, parts, w1, rowmask, eps):
    _chk(x, "x", torch.bfloat16)
    _chk(parts, "parts", torch.float32)
    M, H = x.shape
    _chk_norm(w1, rowmask, M, H)
    S = parts.shape[0]
    if parts.dim() != 3 or parts.shape[1] != M or parts.shape[2] != H:
        raise RuntimeError("parts must be [S, M, H]")
    h, hn = torch.empty_like(x), torch.empty_like(x)
    check(lib().ojx_add_rmsnorm_sk(_ptr(x), _ptr(parts), S, _ptr(w1), _ptr(rowmask), float(eps), _ptr(h), _ptr(hn),
                                   M, H, _stream()))
    return [h, hn]


def add_rmsnorm_sk2(x, parts, w1, rowmask, eps):
    if not 2 <= parts.shape[0] <= 4:
        raise RuntimeError("S must be 2..4")
    return add_rmsnorm_sk(x, parts, w1, rowmask, eps)


def silu_mul(gu):
    _chk(gu, "gu", torch.bfloat16)
    M, I2 = gu.shape
    out = gu.new_empty((M, I2 // 2))
    check(lib().ojx_silu_mul(_ptr(gu), _ptr(out), M, I2 // 2, _stream()))
    return out


def silu_mul_lut(gu, tab):
    _chk(gu, "gu", torch.bfloat16)
    _chk(tab, "tab", torch.bfloat16)
    M, I2 = gu.shape
    out = gu.new_empty((M, I2 // 2))
    check(lib().ojx_silu_mul_lut(_ptr(gu), _ptr(tab), _ptr(out), M, I2 // 2, _stream()))
    return out


def act_tables(like):
    silu_b = torch.empty(65536, dtype=torch.bfloat16, device=like.device)
    sig_f = torch.empty(65536, dtype=torch.float32, device=like.device)
    check(lib().ojx_act_tables(_ptr(silu_b), _ptr(sig_f), _stream()))
    return [silu_b, sig_f]


# ------------------------------------------------------------------------------------------------ projections
def mm(x, w, cfg=None):
    """y = x . w^T, bf16 out (the reference's _mm / lt_matmul / F.linear). w may be a packed weight (pack_weight)."""
    if w.dim() == 4:
        return mm_pk(x, w, cfg)
    _chk(x, "x", torch.bfloat16)
    _chk(w, "w", torch.bfloat16)
    M, K = x.shape
    N = w.shape[0]
    if w.shape[1] != K:
        raise RuntimeError(f"shape mismatch: x {tuple(x.shape)} w {tuple(w.shape)}")
    y = x.new_empty((M, N))
    ws, nws = _workspace(M, N, K, KIND_PLAIN, cfg, x.device)
    check(lib().ojx_gemm_bf16(_ptr(x), _ptr(w), _ptr(y), M, N, K, K, K, N, _ptr(ws), nws, _cfgp(cfg), _stream()))
    return y


def mm_splitk_f32(x, w, S, tile=-1):
    """parts [S, M, N] fp32 over S contiguous K ranges (the reference's _skmm torch.bmm with out_dtype=fp32)."""
    _chk(x, "x", torch.bfloat16)
    _chk(w, "w", torch.bfloat16)
    M, K = x.shape
    N = w.shape[0]
    if w.shape[1] != K:
        raise RuntimeError(f"shape mismatch: x {tuple(x.shape)} w {tuple(w.shape)}")
    parts = torch.empty((S, M, N), dtype=torch.float32, device=x.device)
    check(lib().ojx_gemm_splitk_f32(_ptr(x), _ptr(w), _ptr(parts), M, N, K, K, K, S, tile, _stream()))
    return parts


def mm_silu_mul(x, w_gu_packed, cfg=None):
    """out [M, I] = bf16(bf16(silu(g)) * u), [g | u] = x . W_gu^T, W_gu in pack_gate_up layout [2I, K] (or that
    weight through pack_weight)."""
    if w_gu_packed.dim() == 4:
        return mm_silu_mul_pk(x, w_gu_packed, cfg)
    _chk(x, "x", torch.bfloat16)
    _chk(w_gu_packed, "w_gu", torch.bfloat16)
    M, K = x.shape
    N = w_gu_packed.shape[0]
    if w_gu_packed.shape[1] != K or N % 2:
        raise RuntimeError(f"shape mismatch: x {tuple(x.shape)} w_gu {tuple(w_gu_packed.shape)}")
    out = x.new_empty((M, N // 2))
    ws, nws = _workspace(M, N, K, KIND_SILU_MUL, cfg, x.device)
    check(lib().ojx_gemm_silu_mul(_ptr(x), _ptr(w_gu_packed), _ptr(out), M, N // 2, K, _ptr(ws), nws, _cfgp(cfg),
                                  _stream()))
    return out


def mm_residual_rmsnorm(h, y, w, w1, rowmask, eps, want_hn=True, cfg=None):
    """(h_new, hn): h_new = bf16(h + bf16(y . w^T)); hn = RMSNorm(h_new) * w1 (zero where rowmask == 0). w may be a
    packed weight (pack_weight)."""
    if w.dim() == 4:
        return mm_residual_rmsnorm_pk(h, y, w, w1, rowmask, eps, want_hn, cfg)
    _chk(h, "h", torch.bfloat16)
    _chk(y, "y", torch.bfloat16)
    _chk(w, "w", torch.bfloat16)
    M, K = y.shape
    N = w.shape[0]
    if w.shape[1] != K or tuple(h.shape) != (M, N):
        raise RuntimeError(f"shape mismatch: h {tuple(h.shape)} y {tuple(y.shape)} w {tuple(w.shape)}")
    if want_hn:
        _chk_norm(w1, rowmask, M, N)
    elif rowmask is not None:
        _chk(rowmask, "rowmask", torch.int32)
    h_new = torch.empty_like(h)
    hn = torch.empty_like(h) if want_hn else None
    ws, nws = _workspace(M, N, K, KIND_RESIDUAL, cfg, y.device)
    check(lib().ojx_gemm_residual_rmsnorm(_ptr(y), _ptr(w), _ptr(h), _ptr(w1) if want_hn else None, _ptr(rowmask),
                                          float(eps), _ptr(h_new), _ptr(hn), M, N, K, _ptr(ws), nws, _cfgp(cfg),
                                          _stream()))
    return h_new, hn


def head_scores(hn, lastidx, w, bias=None):
    """scores [R] fp32 = hn[lastidx].float() @ w (+ bias): the scoring head, mdl.head(hn[lastidx].float())
    .squeeze(-1) (src/server.py:37, 57, 129) for a Linear(H, 1) with fp32 weight w [H] (or [1, H]) and bias [1], with
    the row gather fused in. lastidx is int64; an out-of-range index gives NaN for that score."""
    _chk(hn, "hn", torch.bfloat16)
    _chk(lastidx, "lastidx", torch.int64)
    w = w.reshape(-1)
    _chk(w, "w", torch.float32)
    if bias is not None:
        _chk(bias, "bias", torch.float32)
    rows, H = hn.shape
    if w.numel() != H:
        raise RuntimeError(f"w has {w.numel()} elements, hn rows have {H}")
    R = lastidx.numel()
    scores = hn.new_empty(R, dtype=torch.float32)
    check(lib().ojx_head_scores(_ptr(hn), rows, H, _ptr(lastidx), R, _ptr(w), _ptr(bias), _ptr(scores), _stream()))
    return scores


def pack_gate_up(gate, up):
    """W_gu for mm_silu_mul: [2I, K], rows in blocks of 8 (4 gate rows, then the same 4 up rows)."""
    _chk(gate, "gate", torch.bfloat16)
    _chk(up, "up", torch.bfloat16)
    if gate.shape != up.shape:
        raise RuntimeError("gate and up must have the same shape")
    I, K = gate.shape
    packed = torch.empty((2 * I, K), dtype=gate.dtype, device=gate.device)
    check(lib().ojx_pack_gate_up(_ptr(gate), _ptr(up), _ptr(packed), I, K, _stream()))
    return packed


# ------------------------------------------------------------------------------------------------ packed weights
def pack_weight(w):
    """The load-time weight layout of the *_pk projections: W [N, K] -> [K/64, N/16, 16, 64] (ojx_pack_weight). For
    the fused gate-up, pack pack_gate_up's output."""
    _chk(w, "w", torch.bfloat16)
    N, K = w.shape
    if N % 16 or K % 64:
        raise RuntimeError(f"pack_weight needs N % 16 == 0 and K % 64 == 0, got {tuple(w.shape)}")
    wp = torch.empty((K // 64, N // 16, 16, 64), dtype=w.dtype, device=w.device)
    check(lib().ojx_pack_weight(_ptr(w), _ptr(wp), N, K, _stream()))
    return wp


_UNSPLIT = {}   # id(split weight) -> (weak reference to it, its version, its address, W [N, K])


def _unsplit_drop(key):
    def drop(ref):  # the split weight died: forget its W, unless the id already names a newer tensor's entry
        if _UNSPLIT.get(key, (None,))[0] is ref:
            del _UNSPLIT[key]
    return drop


def unsplit_weight(wsk):
    """W [N, K] from the reference's split-K copy wsk [S, K/S, N] (src/fastmodel.py:186-188; ojx_unsplit_weight), for
    callers that hold only that copy (lt2_run / _skmm / _res with a weight from the reference's own _split). The
    result is kept while wsk lives and is made again if wsk is modified in place; during a graph capture it is made
    inside the capture and not kept (the graph's memory pool owns it)."""
    _chk(wsk, "wsk", torch.bfloat16)
    if wsk.dim() != 3:
        raise RuntimeError(f"unsplit_weight: wsk must be [S, K/S, N], got {tuple(wsk.shape)}")
    S, KS, N = wsk.shape
    capturing = torch.cuda.is_current_stream_capturing()
    key = id(wsk)
    hit = None if capturing else _UNSPLIT.get(key)
    if hit is not None and hit[0]() is wsk and hit[1] == wsk._version and hit[2] == wsk.data_ptr():
        return hit[3]
    w = torch.empty((N, S * KS), dtype=wsk.dtype, device=wsk.device)
    check(lib().ojx_unsplit_weight(_ptr(wsk), _ptr(w), N, S * KS, S, _stream()))
    if not capturing:
        _UNSPLIT[key] = (weakref.ref(wsk, _unsplit_drop(key)), wsk._version, wsk.data_ptr(), w)
    return w


def _pk_shape(wp):
    _chk(wp, "wp", torch.bfloat16)
    if wp.dim() != 4 or tuple(wp.shape[2:]) != (16, 64):
        raise RuntimeError(f"a packed weight is [K/64, N/16, 16, 64], got {tuple(wp.shape)}")
    return wp.shape[1] * 16, wp.shape[0] * 64


def mm_pk(x, wp, cfg=None):
    """mm with a packed weight (pack_weight)."""
    _chk(x, "x", torch.bfloat16)
    N, K = _pk_shape(wp)
    M = x.shape[0]
    if x.shape[1] != K:
        raise RuntimeError(f"shape mismatch: x {tuple(x.shape)}, packed weight of K={K}")
    y = x.new_empty((M, N))
    ws, nws = _workspace(M, N, K, KIND_PLAIN | _lib.KIND_PACKED, cfg, x.device)
    check(lib().ojx_gemm_bf16_pk(_ptr(x), _ptr(wp), _ptr(y), M, N, K, K, N, _ptr(ws), nws, _cfgp(cfg), _stream()))
    return y


def mm_silu_mul_pk(x, wgu_pk, cfg=None):
    """mm_silu_mul with the packed gate-up weight (pack_weight(pack_gate_up(gate, up)))."""
    _chk(x, "x", torch.bfloat16)
    N, K = _pk_shape(wgu_pk)
    M = x.shape[0]
    if x.shape[1] != K:
        raise RuntimeError(f"shape mismatch: x {tuple(x.shape)}, packed weight of K={K}")
    out = x.new_empty((M, N // 2))
    ws, nws = _workspace(M, N, K, KIND_SILU_MUL | _lib.KIND_PACKED, cfg, x.device)
    check(lib().ojx_gemm_silu_mul_pk(_ptr(x), _ptr(wgu_pk), _ptr(out), M, N // 2, K, _ptr(ws), nws, _cfgp(cfg),
                                     _stream()))
    return out


def mm_residual_rmsnorm_pk(h, y, wp, w1, rowmask, eps, want_hn=True, cfg=None):
    """mm_residual_rmsnorm with a packed weight."""
    _chk(h, "h", torch.bfloat16)
    _chk(y, "y", torch.bfloat16)
    N, K = _pk_shape(wp)
    M = y.shape[0]
    if y.shape[1] != K or tuple(h.shape) != (M, N):
        raise RuntimeError(f"shape mismatch: h {tuple(h.shape)} y {tuple(y.shape)}, packed weight N={N} K={K}")
    if want_hn:
        _chk_norm(w1, rowmask, M, N)
    elif rowmask is not None:
        _chk(rowmask, "rowmask", torch.int32)
    h_new = torch.empty_like(h)
    hn = torch.empty_like(h) if want_hn else None
    ws, nws = _workspace(M, N, K, KIND_RESIDUAL | _lib.KIND_PACKED, cfg, y.device)
    check(lib().ojx_gemm_residual_rmsnorm_pk(_ptr(y), _ptr(wp), _ptr(h), _ptr(w1) if want_hn else None,
                                             _ptr(rowmask), float(eps), _ptr(h_new), _ptr(hn), M, N, K, _ptr(ws),
                                             nws, _cfgp(cfg), _stream()))
    return h_new, hn


# ------------------------------------------------------------------------------------------------ attention prep
def _prep_outputs(N, HQ, HKV, D, like):
    return (like.new_empty((HQ, N, D)), like.new_empty((HKV, N, D)), like.new_empty((HKV, N, D)),
            like.new_empty((N, HQ * D)))


def _chk_rope(qw1, kw1, cos, sin, N, D):
    """The norm weights are [D] and cos / sin [N, RD] (the kernels read N rows of RD and D weights)."""
    if qw1.numel() != D or kw1.numel() != D:
        raise RuntimeError(f"qw1 and kw1 must have D={D} elements, got {qw1.numel()} and {kw1.numel()}")
    if cos.dim() != 2 or tuple(cos.shape) != tuple(sin.shape) or cos.shape[0] != N:
        raise RuntimeError(f"cos and sin must both be [N={N}, RD], got {tuple(cos.shape)} and {tuple(sin.shape)}")


def fullattn_prep2(proj, qw1, kw1, cos, sin, B, T, HQ, HKV, D, eps):
    """The reference extension's fullattn_prep2 (src/kernels.cu:302-360) for B = 1 (the tree forward's call,
    src/fastmodel.py:462): [qt [1, HQ, T, D], kt [1, HKV, T, D], vt [1, HKV, T, D], gate [T, HQ D]]."""
    _chk(proj, "proj", torch.bfloat16)
    _chk(qw1, "qw1", torch.float32)
    _chk(kw1, "kw1", torch.float32)
    _chk(cos, "cos", torch.bfloat16)
    _chk(sin, "sin", torch.bfloat16)
    if B != 1:
        raise RuntimeError("fullattn_prep2: B must be 1 (the packed-token forward)")
    N = proj.shape[0]
    if N != T or proj.shape[1] != (2 * HQ + 2 * HKV) * D:
        raise RuntimeError(f"proj {tuple(proj.shape)} does not match T={T}, HQ={HQ}, HKV={HKV}, D={D}")
    _chk_rope(qw1, kw1, cos, sin, N, D)
    RD = cos.shape[1]
    qt, kt, vt, gate = _prep_outputs(N, HQ, HKV, D, proj)
    check(lib().ojx_fullattn_prep(_ptr(proj), N, HQ, HKV, D, RD, float(eps), _ptr(qw1), _ptr(kw1), _ptr(cos),
                                  _ptr(sin), _ptr(qt), _ptr(kt), _ptr(vt), _ptr(gate), _stream()))
    return [qt.unsqueeze(0), kt.unsqueeze(0), vt.unsqueeze(0), gate]


def linattn_prep_dedup2(proj, hist, rep_ptr, rep_pos, L2, convw, A_log, dt_bias, KD, VD, HV, HK, HD, rep_qk):
    """The reference extension's linattn_prep_dedup2 (src/kernels.cu:1176-1290), as forward_gtree calls it
    (src/fastmodel.py:420,438): [q [R, RQ KD], k, v [R, VD], g fp32 [R, HV], beta [R, HV]], R = rep_pos.numel(),
    RQ = HV / HK when rep_qk else 1."""
    _chk(proj, "proj", torch.bfloat16)
    for t, nm in ((hist, "hist"), (rep_ptr, "rep_ptr"), (rep_pos, "rep_pos")):
        _chk(t, nm, torch.int32)
    for t, nm in ((convw, "convw"), (A_log, "A_log"), (dt_bias, "dt_bias")):
        _chk(t, nm, torch.bfloat16)
    N, R = proj.shape[0], rep_pos.numel()
    C = 2 * KD + VD
    if proj.dim() != 2 or proj.shape[1] != C + VD + 2 * HV:
        raise RuntimeError(f"proj {tuple(proj.shape)} is not [N, 2 KD + 2 VD + 2 HV] for KD={KD} VD={VD} HV={HV}")
    if convw.numel() != C * 4 or (convw.dim() == 2 and convw.shape[1] != 4):
        raise RuntimeError(f"convw {tuple(convw.shape)} is not [{C}, 4]")
    if hist.numel() != (N + 1) * 4 or rep_ptr.numel() != N + 2 or A_log.numel() != HV or dt_bias.numel() != HV:
        raise RuntimeError("hist must be [N + 1, 4], rep_ptr [N + 2], A_log and dt_bias [HV]")
    rq = HV // HK if rep_qk else 1
    q, k, v = proj.new_empty((R, rq * KD)), proj.new_empty((R, rq * KD)), proj.new_empty((R, VD))
    g, beta = proj.new_empty((R, HV), dtype=torch.float32), proj.new_empty((R, HV))
    check(lib().ojx_linattn_prep(_ptr(proj), _ptr(hist), _ptr(rep_ptr), _ptr(rep_pos), N, R, int(L2), _ptr(convw),
                                 _ptr(A_log), _ptr(dt_bias), KD, VD, HV, HK, HD, int(bool(rep_qk)), _ptr(q), _ptr(k),
                                 _ptr(v), _ptr(g), _ptr(beta), _stream()))
    return [q, k, v, g, beta]


def mm_fullattn_prep(x, w_qkv, qw1, kw1, cos, sin, HQ, HKV, D, eps, fused=False):
    """_mm(hn, d.w_in) + fullattn_prep2 (src/fastmodel.py:412,462): the QKV in-projection and the full-attention
    prep. w_qkv row-major [(2 HQ + 2 HKV) D, K] or packed (pack_weight). Returns the prep's outputs
    [qt [1, HQ, M, D], kt, vt, gate [M, HQ D]]. By default the planned GEMM followed by the prep kernel (two
    launches, the faster route at every measured M); fused=True runs ojx_gemm_qkv_fullattn_prep, the prep in the
    GEMM's epilogue (one launch, the [M, (2 HQ + 2 HKV) D] projection never stored)."""
    if not fused:
        rows = _pk_shape(w_qkv)[0] if w_qkv.dim() == 4 else w_qkv.shape[0]
        if rows != (2 * HQ + 2 * HKV) * D:
            raise RuntimeError(f"w_qkv does not match x {tuple(x.shape)}, HQ={HQ}, HKV={HKV}, D={D}")
        return fullattn_prep2(mm(x, w_qkv), qw1, kw1, cos, sin, 1, x.shape[0], HQ, HKV, D, eps)
    _chk(x, "x", torch.bfloat16)
    for t, nm in ((qw1, "qw1"), (kw1, "kw1")):
        _chk(t, nm, torch.float32)
    _chk(cos, "cos", torch.bfloat16)
    _chk(sin, "sin", torch.bfloat16)
    M, K = x.shape
    packed = w_qkv.dim() == 4
    N, Kw = _pk_shape(w_qkv) if packed else tuple(w_qkv.shape)
    if Kw != K or N != (2 * HQ + 2 * HKV) * D:
        raise RuntimeError(f"w_qkv does not match x {tuple(x.shape)}, HQ={HQ}, HKV={HKV}, D={D}")
    _chk_rope(qw1, kw1, cos, sin, M, D)
    qt, kt, vt, gate = _prep_outputs(M, HQ, HKV, D, x)
    check(lib().ojx_gemm_qkv_fullattn_prep(_ptr(x), _ptr(w_qkv), int(packed), _ptr(qw1), _ptr(kw1), _ptr(cos),
                                           _ptr(sin), _ptr(qt), _ptr(kt), _ptr(vt), _ptr(gate), M, K, HQ, HKV, D,
                                           cos.shape[1], float(eps), _stream()))
    return [qt.unsqueeze(0), kt.unsqueeze(0), vt.unsqueeze(0), gate]


# ------------------------------------------------------------------------------------------------ attention cores
def _one_device(*tensors):
    """The launches go on the current device's stream: every tensor has to live there."""
    cur = torch._C._cuda_getDevice()
    for t in tensors:
        if t is not None and t.get_device() != cur:
            raise RuntimeError(f"all tensors must be on the current device cuda:{cur}, got {t.device}")


def _scratch(n, like):
    """Workspace of one call, from torch's allocator: ordered on the current stream, and in a graph capture part of the
    graph's own memory, so that no two graphs or streams share it."""
    return torch.empty(n, dtype=torch.uint8, device=like.device) if n > 0 else None


def _heads_rows(t, name):
    """(heads, rows, D) of a prep output, [heads, N, D] or with the leading batch axis of 1."""
    _chk(t, name, torch.bfloat16)
    if t.dim() == 4 and t.shape[0] == 1:
        return t.shape[1:]
    if t.dim() != 3:
        raise RuntimeError(f"{name} must be [heads, N, D] or [1, heads, N, D], got {tuple(t.shape)}")
    return t.shape


def _chk_cache(kc, vc, ks, vs, HKV, D):
    """(format, pages, page) of a paged cache."""
    fmt = {torch.bfloat16: _lib.KV_BF16, torch.float8_e4m3fn: _lib.KV_E4M3}.get(kc.dtype)
    if fmt is None:
        raise RuntimeError(f"a cache is torch.bfloat16 or torch.float8_e4m3fn, got {kc.dtype}")
    _chk(kc, "kc")
    _chk(vc, "vc", kc.dtype)
    if kc.dim() != 4 or kc.shape != vc.shape or kc.shape[1] != HKV or kc.shape[3] != D:
        raise RuntimeError(f"kc {tuple(kc.shape)} and vc {tuple(vc.shape)} must both be [pages, HKV={HKV}, page, D={D}]")
    if fmt == _lib.KV_E4M3:
        _chk(ks, "ks", torch.float32)
        _chk(vs, "vs", torch.float32)
        if ks.shape != kc.shape[:3] or vs.shape != kc.shape[:3]:
            raise RuntimeError(f"ks {tuple(ks.shape)} and vs {tuple(vs.shape)} must be {tuple(kc.shape[:3])}")
    elif ks is not None or vs is not None:
        raise RuntimeError("a bf16 cache has no scales")
    return fmt, kc.shape[0], kc.shape[2]


def kv_cache_write(k, v, slots, kc, vc, ks=None, vs=None):
    """Writes N tokens' keys and values into a paged cache, in place. k, v bf16 [HKV, N, D] (fullattn_prep2's kt and vt,
    with or without their batch axis); slots int64 [N], page index * page + place (outside the cache: not written); kc, vc
    [pages, HKV, page, D], bf16, or float8_e4m3fn with the rows' scales ks, vs fp32 [pages, HKV, page]. The e4m3 form
    stores x / scale with scale the smallest power of two that brings the row within +-448. Two tokens with one slot leave a
    mixture of both there."""
    HKV, N, D = _heads_rows(k, "k")
    if tuple(_heads_rows(v, "v")) != (HKV, N, D):
        raise RuntimeError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must have one shape")
    fmt, pages, page = _chk_cache(kc, vc, ks, vs, HKV, D)
    _chk(slots, "slots", torch.int64)
    if slots.numel() != N:
        raise RuntimeError(f"slots must have N={N} elements, got {slots.numel()}")
    _one_device(k, v, slots, kc, vc, ks, vs)
    check(lib().ojx_kv_cache_write(_ptr(k), _ptr(v), _ptr(slots), N, HKV, D, fmt, _ptr(kc), _ptr(vc), _ptr(ks), _ptr(vs),
                                   pages, page, _stream()))


def kv_cache_read(kc, vc, slots, ks=None, vs=None):
    """(k, v) bf16 [HKV, N, D]: the tokens in slots int64 [N] of a paged cache (see kv_cache_write), zeros for a slot
    outside it."""
    if kc.dim() != 4:
        raise RuntimeError(f"kc must be [pages, HKV, page, D], got {tuple(kc.shape)}")
    HKV, D = kc.shape[1], kc.shape[3]
    fmt, pages, page = _chk_cache(kc, vc, ks, vs, HKV, D)
    _chk(slots, "slots", torch.int64)
    N = slots.numel()
    _one_device(slots, kc, vc, ks, vs)
    k = slots.new_empty((HKV, N, D), dtype=torch.bfloat16)
    v = torch.empty_like(k)
    check(lib().ojx_kv_cache_read(_ptr(kc), _ptr(vc), _ptr(ks), _ptr(vs), _ptr(slots), N, HKV, D, fmt, _ptr(k), _ptr(v),
                                  pages, page, _stream()))
    return k, v


def tree_bits(parents):
    """The bits that tree_attn takes, int64 [N, words] on the CPU, for sequences of drafted tokens given by their parents:
    parents[b][j] is the index within sequence b of token j's parent, smaller than j, or -1 for a token that follows the
    context. A token sees its ancestors and itself."""
    words = max([1] + [-(-len(p) // 64) for p in parents])
    rows = []
    for b, p in enumerate(parents):
        seen = []
        for j, parent in enumerate(p):
            parent = int(parent)
            if not -1 <= parent < j:
                raise RuntimeError(f"parents[{b}][{j}] = {parent} must be -1 or the index of an earlier token")
            seen.append((seen[parent] if parent >= 0 else 0) | 1 << j)
        rows += seen
    flat = [(x >> 64 * w) & ((1 << 64) - 1) for x in rows for w in range(words)]
    return torch.tensor([x - (1 << 64) if x >> 63 else x for x in flat], dtype=torch.int64).reshape(len(rows), words)


def tree_attn(q, kc, vc, table, ctx, q_ptr, bits=None, ks=None, vs=None, scale=None, want_lse=False):
    """Attention of drafted tokens over a paged cache: out bf16 [N, HQ D], with want_lse (out, lse fp32 [N, HQ]).
    q bf16 [HQ, N, D] (fullattn_prep2's qt, with or without its batch axis); the cache as in kv_cache_write; table int32
    [B, max_pages], ctx int32 [B], q_ptr int32 [B + 1]. Sequence b's query rows are q_ptr[b] .. q_ptr[b+1] - 1, its
    drafted tokens; drafted token j stands in the cache at position ctx[b] + j, written before this call. A row sees the
    ctx[b] positions before the drafted tokens, and those drafted tokens whose bit is set in its bits int64 [N, words]
    (tree_bits); with bits=None its predecessors and itself (a plain continuation, or a single token). A row that sees
    nothing, or belongs to no sequence, gives zeros (lse -inf). scale defaults to D ** -0.5."""
    HQ, N, D = _heads_rows(q, "q")
    if kc.dim() != 4 or kc.shape[1] < 1 or HQ % kc.shape[1]:
        raise RuntimeError(f"kc {tuple(kc.shape)} must be [pages, HKV, page, D] with HKV dividing HQ={HQ}")
    HKV = kc.shape[1]
    fmt, pages, page = _chk_cache(kc, vc, ks, vs, HKV, D)
    for t, nm in ((table, "table"), (ctx, "ctx"), (q_ptr, "q_ptr")):
        _chk(t, nm, torch.int32)
    B = ctx.numel()
    if table.dim() != 2 or table.shape[0] != B or q_ptr.numel() != B + 1:
        raise RuntimeError(f"table {tuple(table.shape)} must be [B={B}, max_pages] and q_ptr [B + 1], got "
                           f"{q_ptr.numel()}")
    words = 0
    if bits is not None:
        _chk(bits, "bits", torch.int64)
        if bits.dim() != 2 or bits.shape[0] != N or bits.shape[1] < 1:
            raise RuntimeError(f"bits must be [N={N}, words], got {tuple(bits.shape)}")
        words = bits.shape[1]
    _one_device(q, kc, vc, ks, vs, table, ctx, q_ptr, bits)
    out = q.new_empty((N, HQ * D))
    lse = q.new_empty((N, HQ), dtype=torch.float32) if want_lse else None
    MP = table.shape[1]
    n = lib().ojx_tree_attn_workspace(N, B, HQ, HKV, D, MP, page)
    if n < 0:
        check(2)
    ws = _scratch(n, q)
    check(lib().ojx_tree_attn(_ptr(q), _ptr(q_ptr), _ptr(ctx), _ptr(bits), words, _ptr(kc), _ptr(vc), _ptr(ks), _ptr(vs),
                              fmt, _ptr(table), MP, N, B, HQ, HKV, D, pages, page,
                              float(D ** -0.5 if scale is None else scale), _ptr(out), _ptr(lse), _ptr(ws), n,
                              _stream()))
    return (out, lse) if want_lse else out


def _chk_linattn(q, k, v, g, beta):
    """(R, HV, HK) of the linear-attention operands (linattn_prep_dedup2's outputs)."""
    _chk(q, "q", torch.bfloat16)
    _chk(k, "k", torch.bfloat16)
    _chk(v, "v", torch.bfloat16)
    _chk(g, "g", torch.float32)
    if q.dim() != 2 or q.shape != k.shape or q.shape[1] % 128 or q.shape[1] == 0:
        raise RuntimeError(f"q {tuple(q.shape)} and k {tuple(k.shape)} must both be [R, HK 128]")
    R, HK = q.shape[0], q.shape[1] // 128
    if g.dim() != 2 or g.shape[0] != R:
        raise RuntimeError(f"g must be [R={R}, HV], got {tuple(g.shape)}")
    HV = g.shape[1]
    if tuple(v.shape) != (R, HV * 128) or HV % HK or HV == 0:
        raise RuntimeError(f"v {tuple(v.shape)} must be [R={R}, HV 128] with HV={HV} a multiple of HK={HK}")
    if beta is not None:
        _chk(beta, "beta", torch.bfloat16)
        if beta.shape != g.shape:
            raise RuntimeError(f"beta {tuple(beta.shape)} must be [R, HV] = {tuple(g.shape)}")
    return R, HV, HK


def _chk_states(state, HV):
    _chk(state, "state", torch.float32)
    if state.dim() != 4 or tuple(state.shape[1:]) != (HV, 128, 128):
        raise RuntimeError(f"state must be [slots, HV={HV}, 128, 128], got {tuple(state.shape)}")


def linattn_prompt(q, k, v, g, beta, seq_ptr, state=None, src=None, scale=None):
    """Linear attention with a decay for each head over whole sequences, on linattn_prep_dedup2's outputs:
    (o bf16 [R, HV 128], states fp32 [S, HV, 128, 128]). q, k bf16 [R, HK 128], v bf16 [R, HV 128], g fp32 [R, HV] (the
    decay's logarithm), beta bf16 [R, HV], or None for plain decayed sums without the delta rule. Sequence s is rows
    seq_ptr[s] .. seq_ptr[s+1] - 1 (int32 [S + 1]; the path slots of the tree layout: seq_ptr = arange(0, R + 1, L2)).
    It starts from state[src[s]] (state fp32 [slots, HV, 128, 128], src int32 [S], -1 = zeros; src=None: state[s];
    state=None: zeros), so that paths can go on from a state that they share. scale defaults to 128 ** -0.5."""
    R, HV, HK = _chk_linattn(q, k, v, g, beta)
    _chk(seq_ptr, "seq_ptr", torch.int32)
    S = seq_ptr.numel() - 1
    if S < 0:
        raise RuntimeError("seq_ptr must be [S + 1]")
    slots = 0
    if state is not None:
        _chk_states(state, HV)
        slots = state.shape[0]
        if src is None and slots != S:
            raise RuntimeError(f"without src there must be S={S} states, got {slots}")
    if src is not None:
        if state is None:
            raise RuntimeError("src without state")
        _chk(src, "src", torch.int32)
        if src.numel() != S:
            raise RuntimeError(f"src must have S={S} elements, got {src.numel()}")
    _one_device(q, k, v, g, beta, seq_ptr, state, src)
    o = torch.empty_like(v)
    last = q.new_empty((S, HV, 128, 128), dtype=torch.float32)
    n = lib().ojx_linattn_prompt_workspace(R, S, HV, HK, beta is not None)
    if n < 0:
        check(2)
    ws = _scratch(n, q)
    # a pool of no states has no address, and none stands for zeros: any other, which 0 slots keep from being read
    at = _ptr(last if state is not None and slots == 0 else state)
    check(lib().ojx_linattn_prompt(_ptr(q), _ptr(k), _ptr(v), _ptr(g), _ptr(beta), _ptr(seq_ptr), at, _ptr(src),
                                   slots, R, S, HV, HK, float(128 ** -0.5 if scale is None else scale), _ptr(o),
                                   _ptr(last), _ptr(ws), n, _stream()))
    return o, last


def linattn_step(q, k, v, g, beta, state, slot, scale=None):
    """linattn_prompt for single tokens: o bf16 [R, HV 128]; row r's token runs on state[slot[r]] (state fp32 [slots, HV,
    128, 128], slot int32 [R]), which is updated in place. A negative slot is an idle row (zeros); a slot that is not in
    state, or that an earlier row names too, gives NaN and no update. Operands as in linattn_prompt."""
    R, HV, HK = _chk_linattn(q, k, v, g, beta)
    _chk_states(state, HV)
    _chk(slot, "slot", torch.int32)
    if slot.numel() != R:
        raise RuntimeError(f"slot must have R={R} elements, got {slot.numel()}")
    _one_device(q, k, v, g, beta, state, slot)
    o = torch.empty_like(v)
    check(lib().ojx_linattn_step(_ptr(q), _ptr(k), _ptr(v), _ptr(g), _ptr(beta), _ptr(state), _ptr(slot), state.shape[0],
                                 R, HV, HK, float(128 ** -0.5 if scale is None else scale), _ptr(o), _stream()))
    return o


# ------------------------------------------------------------------------------------------------ drafted tokens
def _chk_each(*named):
    """_chk of (tensor, name, dtype) one after the other, without a call for each that is as it should be."""
    for t, name, dtype in named:
        if t is None or not t.is_cuda or t.dtype is not dtype or not t.is_contiguous():
            _chk(t, name, dtype)


@functools.lru_cache(1024)
def _work_bytes(name, *sizes):
    """The library's answer to how much workspace calls of these sizes need."""
    n = getattr(lib(), name)(*sizes)
    if n < 0:
        check(2)
    return n


def _chk_count(t, name, n):
    if t.numel() != n:
        raise RuntimeError(f"{name} must have {n} elements, got {t.numel()}")


def _chk_rows(q_ptr, N, *counted):
    """B of the sequences that q_ptr int32 [B + 1] makes of N rows; counted: (tensor, name, one each of N rows?)."""
    B = q_ptr.numel() - 1
    if B < 0:
        raise RuntimeError("q_ptr must be [B + 1]")
    for t, name, rows in counted:
        _chk_count(t, name, N if rows else B)
    return B


def _chk_slots(state, slot, HV, B):
    _chk_states(state, HV)
    _chk_each((slot, "slot", torch.int32))
    _chk_count(slot, "slot", B)


def linattn_tree(q, k, v, g, beta, state, slot, q_ptr, parents=None, scale=None):
    """linattn_step for drafted tokens, a tree of them or a line: o bf16 [N, HV 128], on states that stay as they are.
    Sequence b's rows are q_ptr[b] .. q_ptr[b+1] - 1 (int32 [B + 1]), its state is state[slot[b]] (fp32 [slots, HV, 128,
    128], int32 [B]). Row j of a sequence follows its row parents[j] (int32 [N], indexes within the sequence), or the state
    itself where parents[j] is not one of 0 .. j - 1; parents=None: each row follows the one before it. A row's output is that
    of its path's tokens, from the state on. A negative slot gives zeros, a slot that is not in state NaN; a row of no sequence gives
    zeros. Operands as in linattn_prompt. linattn_keep then takes the states over the tokens that are kept."""
    N, HV, HK = _chk_linattn(q, k, v, g, beta)
    _chk_each((q_ptr, "q_ptr", torch.int32))
    B = _chk_rows(q_ptr, N)
    if parents is not None:
        _chk_each((parents, "parents", torch.int32))
        _chk_count(parents, "parents", N)
    _chk_slots(state, slot, HV, B)
    _one_device(q, k, v, g, beta, state, slot, q_ptr, parents)
    o = torch.empty_like(v)
    n = _work_bytes("ojx_linattn_tree_workspace", N, B, HV, HK)
    ws = _scratch(n, q)
    check(lib().ojx_linattn_tree(_ptr(q), _ptr(k), _ptr(v), _ptr(g), _ptr(beta), _ptr(state), _ptr(slot), state.shape[0],
                                 _ptr(q_ptr), _ptr(parents), N, B, HV, HK, float(128 ** -0.5 if scale is None else scale),
                                 _ptr(o), _ptr(ws), n, _stream()))
    return o


def linattn_keep(k, v, g, beta, state, slot, q_ptr, path, count):
    """Takes states forward over the tokens that were kept, in place: state[slot[b]] over sequence b's rows path[q_ptr[b] +
    i], i < count[b], one after the other (path int32 [N] and count int32 [B] as verify_drafts gives them; the other
    operands as linattn_tree took them). A slot that is not in state, or that an earlier sequence has too, is left alone."""
    N, HV, HK = _chk_linattn(k, k, v, g, beta)
    _chk_each((q_ptr, "q_ptr", torch.int32), (path, "path", torch.int32), (count, "count", torch.int32))
    B = _chk_rows(q_ptr, N, (path, "path", True), (count, "count", False))
    _chk_slots(state, slot, HV, B)
    _one_device(k, v, g, beta, state, slot, q_ptr, path, count)
    check(lib().ojx_linattn_keep(_ptr(k), _ptr(v), _ptr(g), _ptr(beta), _ptr(state), _ptr(slot), state.shape[0], _ptr(q_ptr),
                                 _ptr(path), _ptr(count), N, B, HV, HK, _stream()))


def _chk_vocab(t, name, N=None, V=None):
    """(type, N, V, row stride) of logits or probabilities: rows may be further apart than they are long."""
    kind = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}.get(t.dtype)
    if kind is None:
        raise RuntimeError(f"{name} must be torch.float32 or torch.bfloat16, got {t.dtype}")
    if not t.is_cuda or t.dim() != 2 or t.shape[1] < 1 or (t.shape[1] > 1 and t.stride(1) != 1):
        raise RuntimeError(f"{name} must be CUDA [N, V] with contiguous rows, got {tuple(t.shape)}")
    if N is not None and tuple(t.shape) != (N, V):
        raise RuntimeError(f"{name} must be [N={N}, V={V}], got {tuple(t.shape)}")
    ld = t.stride(0) if t.shape[0] > 1 else t.shape[1]
    if ld < t.shape[1]:
        raise RuntimeError(f"{name} has rows that overlap")
    return kind, t.shape[0], t.shape[1], ld


def verify_drafts(logits, tokens, q_ptr, u, parents=None, probs=None, temperature=None):
    """Drafted tokens accepted or not, from given random numbers, so that what comes out is distributed as the target's own
    tokens: (path int32 [N], count int32 [B], next int64 [B]).

    Sequence b's rows are q_ptr[b] .. q_ptr[b+1] - 1 (int32 [B + 1]): row 0 is its last token, row j >= 1 the drafted token
    tokens[j] (int64 [N]) behind row parents[j] (int32 [N], within the sequence; None: the row before it). logits [N, V],
    fp32 or bf16 (rows may have a stride): row j's are the target's behind token j. temperature fp32 [B], or None for 1; 0
    takes the first largest logit. probs [N, V], fp32 or bf16: row j's is the distribution that the tokens behind row j were
    drawn from, each by itself; None: they were certain (looked up). u fp32 [N] in [0, 1): row j's number tests its token,
    row 0's draws the next one.

    path has each sequence's accepted rows in order, row 0 first, and -1 behind them; count says how many, next is the token
    behind the last of them (-1: its logits are no distribution, or the sequence has no rows). kv_cache_keep and
    linattn_keep take path and count as they are."""
    kind, N, V, ldl = _chk_vocab(logits, "logits")
    _chk_each((tokens, "tokens", torch.int64), (u, "u", torch.float32), (q_ptr, "q_ptr", torch.int32))
    B = _chk_rows(q_ptr, N, (tokens, "tokens", True), (u, "u", True))
    if parents is not None:
        _chk_each((parents, "parents", torch.int32))
        _chk_count(parents, "parents", N)
    pkind, ldp = 0, 0
    if probs is not None:
        pkind, _, _, ldp = _chk_vocab(probs, "probs", N, V)
    if temperature is not None:
        _chk_each((temperature, "temperature", torch.float32))
        _chk_count(temperature, "temperature", B)
    _one_device(logits, tokens, q_ptr, u, parents, probs, temperature)
    path, count = q_ptr.new_empty(N), q_ptr.new_empty(B)
    token = tokens.new_empty(B)
    n = _work_bytes("ojx_verify_drafts_workspace", N, B, V, probs is not None)
    ws = _scratch(n, logits)
    check(lib().ojx_verify_drafts(_ptr(logits), kind, ldl, _ptr(tokens), _ptr(q_ptr), _ptr(u), _ptr(parents), _ptr(probs),
                                  pkind, ldp, _ptr(temperature), N, B, V, _ptr(path), _ptr(count), _ptr(token), _ptr(ws), n,
                                  _stream()))
    return path, count, token


_CACHE = {torch.bfloat16: _lib.KV_BF16, torch.float8_e4m3fn: _lib.KV_E4M3}


def _chk_layers(kc, vc, ks, vs):
    """(format, layers, pages, HKV, page, D) of a cache [pages, HKV, page, D], or of several layers' [layers, pages, ..]."""
    fmt, shape = _CACHE.get(kc.dtype), kc.shape
    if fmt is None:
        raise RuntimeError(f"a cache is torch.bfloat16 or torch.float8_e4m3fn, got {kc.dtype}")
    _chk_each((kc, "kc", kc.dtype), (vc, "vc", kc.dtype))
    if len(shape) not in (4, 5) or vc.shape != shape:
        raise RuntimeError(f"kc {tuple(shape)} and vc {tuple(vc.shape)} must both be [pages, HKV, page, D], or [layers, pages, "
                           "HKV, page, D]")
    if fmt == _lib.KV_E4M3:
        _chk_each((ks, "ks", torch.float32), (vs, "vs", torch.float32))
        if ks.shape != shape[:-1] or vs.shape != shape[:-1]:
            raise RuntimeError(f"ks {tuple(ks.shape)} and vs {tuple(vs.shape)} must be {tuple(shape[:-1])}")
    elif ks is not None or vs is not None:
        raise RuntimeError("a bf16 cache has no scales")
    return (fmt, 1, *shape) if len(shape) == 4 else (fmt, *shape)


def _chk_table(table, B=None):
    _chk_each((table, "table", torch.int32))
    shape = table.shape
    if len(shape) != 2 or (B is not None and shape[0] != B):
        raise RuntimeError(f"table {tuple(shape)} must be [B{'' if B is None else '=' + str(B)}, max_pages]")
    return shape


def kv_cache_keep(kc, vc, table, ctx, q_ptr, path, count, ks=None, vs=None):
    """Moves the kept tokens' keys and values together, in place: sequence b's row at position ctx[b] + path[q_ptr[b] + i]
    goes to ctx[b] + i, i < count[b] (path and count as verify_drafts gives them, ctx, table and q_ptr as tree_attn takes
    them). The cache as in kv_cache_write, or that of several layers with one table: [layers, pages, HKV, page, D], scales
    [layers, pages, HKV, page]. Add count to ctx afterwards."""
    fmt, layers, pages, HKV, page, D = _chk_layers(kc, vc, ks, vs)
    _chk_each((q_ptr, "q_ptr", torch.int32), (path, "path", torch.int32), (count, "count", torch.int32),
              (ctx, "ctx", torch.int32))
    N = path.numel()
    B = _chk_rows(q_ptr, N, (count, "count", False), (ctx, "ctx", False))
    MP = _chk_table(table, B)[1]
    _one_device(kc, vc, ks, vs, table, ctx, q_ptr, path, count)
    check(lib().ojx_kv_cache_keep(_ptr(kc), _ptr(vc), _ptr(ks), _ptr(vs), fmt, layers, pages, HKV, page, D, _ptr(table), MP,
                                  _ptr(ctx), _ptr(q_ptr), _ptr(path), _ptr(count), N, B, _stream()))


def _pages_call(table, refs, per_slot, name):
    B, MP = _chk_table(table)
    _chk_each((refs, "refs", torch.int32), (per_slot, name, torch.int32))
    _chk_count(per_slot, name, B)
    return B, MP, refs.numel()


def kv_pages_resize(table, refs, tokens, page):
    """Gives every sequence the pages that tokens[b] tokens need (int32 [B]; negative: left as it is), in place: table int32
    [B, max_pages], refs int32 [pages] = how many table entries name each page. Entries behind that are given back (-1),
    entries that name no page get the lowest free ones, sequence by sequence. tokens[b] = 0 frees a sequence. Returns missing
    int32 [B]: entries for which the pool or the table had no room."""
    B, MP, pages = _pages_call(table, refs, tokens, "tokens")
    _one_device(table, refs, tokens)
    missing = table.new_empty(B)
    n = _work_bytes("ojx_kv_pages_workspace", B, MP, pages, 0)
    ws = _scratch(n, table)
    check(lib().ojx_kv_pages_resize(_ptr(table), MP, _ptr(refs), pages, _ptr(tokens), B, page, _ptr(missing), _ptr(ws), n,
                                    _stream()))
    return missing


def kv_pages_fork(table, ctx, refs, src, page):
    """Slot b's sequence becomes a copy of slot src[b]'s (int32 [B]; b itself: left as it is; outside 0 .. B - 1: empty), in
    place and all at once: full pages are shared, a last page that is not full is taken anew. Returns pairs int32 [B, 2], the
    pages to copy: kv_pages_copy does that for a layer or several, and has to before anything else writes to the cache or
    takes pages. A slot for which the pool has no page left ends with its last full page (its ctx says so)."""
    B, MP, pages = _pages_call(table, refs, src, "src")
    _chk_each((ctx, "ctx", torch.int32))
    _chk_count(ctx, "ctx", B)
    _one_device(table, ctx, refs, src)
    pairs = table.new_empty((B, 2))
    n = _work_bytes("ojx_kv_pages_workspace", B, MP, pages, 1)
    ws = _scratch(n, table)
    check(lib().ojx_kv_pages_fork(_ptr(table), MP, _ptr(ctx), _ptr(refs), pages, _ptr(src), B, page, _ptr(pairs), _ptr(ws),
                                  n, _stream()))
    return pairs


def kv_pages_copy(kc, vc, pairs, ks=None, vs=None):
    """Copies page pairs[i][0] to page pairs[i][1] (int32 [n, 2], as kv_pages_fork gives them; a pair with a page outside the
    cache is left out) in a cache of one layer or several (see kv_cache_keep). No page may be both read and written, or written
    twice."""
    fmt, layers, pages, HKV, page, D = _chk_layers(kc, vc, ks, vs)
    _chk_each((pairs, "pairs", torch.int32))
    if pairs.dim() != 2 or pairs.shape[1] != 2:
        raise RuntimeError(f"pairs must be [n, 2], got {tuple(pairs.shape)}")
    _one_device(kc, vc, ks, vs, pairs)
    check(lib().ojx_kv_pages_copy(_ptr(kc), _ptr(vc), _ptr(ks), _ptr(vs), fmt, layers, pages, HKV, page, D, _ptr(pairs),
                                  pairs.shape[0], _stream()))
