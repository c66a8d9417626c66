"""torch-tensor front end of the gfx950 kernels.

Operator surface kept from the reference:
  ours_flash(q, k, v, sel_idx, exp_idx, kbar, vbar, log_n, nb=None)      methods_eager.py:161-172
  decode_expand_attention(q, k, v, sel_idx, exp_idx, kbar, vbar, log_n,
                          sm_scale=None, block_n=64, block_b=64, num_warps=4)
                                                                        triton_expand_decode.py:139-165
plus one function per decode stage (index_update, qgs_prep, qgs_scan, topk_select, errorgate,
waterfill, topq, residual, residual_flash, dense_decode) and the operators of the 4-bit paged cache
(qk_norm_rope, kv_pages_extend, kv_pages_truncate, kv4_write, kv4_read, kv4_attn), each a thin checked
call of the C ABI (include/openattention_amd.h) on torch's current HIP stream.  Shape, dtype, device, alignment
and stride checks happen here; the kernels trust them.  There is no CPU path: tensors must live
on a HIP device and the kernel library must be built.
"""
from __future__ import annotations

import functools
from operator import index

import numpy as np
import torch
from torch.overrides import _get_current_function_mode_stack
from torch.utils._device import DeviceContext

from openattention_amd import lib

HEAD_DIM = 128
RANK_Q = 32
RANK_C = 16
GROUP = 4


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def _stream(dev: torch.device):
    return torch.cuda.current_stream(dev).cuda_stream


def _dev(*ts: torch.Tensor) -> torch.device:
    dev = None
    for t in ts:
        if t is None:
            continue
        if t.device.type != "cuda":
            raise RuntimeError("openattention_amd kernels need tensors on a HIP device "
                               f"(got {t.device}); there is no CPU fallback")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise RuntimeError(f"tensors on different devices: {dev} and {t.device}")
    return dev


def _on(dev: torch.device, *ts: torch.Tensor) -> None:
    """_dev's checks of further tensors against the device it returned (by index: a step checks 30 of
    them, on the host path of every eager call)."""
    i = dev.index
    for t in ts:
        if t is not None and t.get_device() != i:
            _dev(t)
            raise RuntimeError(f"tensors on different devices: {dev} and {t.device}")


def _need(cond: bool, msg: str) -> None:
    if not cond:
        raise ValueError(msg)


def _chk(t: torch.Tensor, name: str, dtype: torch.dtype, shape: tuple | None = None,
         contiguous: bool = False) -> None:
    """dtype, exact shape (None entries: any extent; a negative entry -m: at least m) and, when
    asked, contiguity -- the layout the kernels index without further checks."""
    _need(t.dtype == dtype, f"{name}: dtype must be {dtype} (got {t.dtype})")
    if shape is not None:
        ok = t.dim() == len(shape) and all(
            want is None or (got == want if want >= 0 else got >= -want)
            for got, want in zip(t.shape, shape))
        _need(ok, f"{name}: shape {tuple(t.shape)} does not match {shape} (-m: at least m)")
    if contiguous:
        _need(t.is_contiguous(), f"{name}: must be contiguous")
    else:
        _need(t.dim() == 0 or t.stride(-1) == 1, f"{name}: last dimension must be contiguous")


def _stats(R: int, C: int, *named) -> None:
    """pooled statistics (R, C, 128) fp32, contiguous (the kernels step rows by C * 128)"""
    for t, name in named:
        _chk(t, name, torch.float32, (R, C, HEAD_DIM), contiguous=True)


def _rows_contig(t: torch.Tensor, name: str, align_elems: int = 1) -> None:
    _need(t.stride(-1) == 1, f"{name}: last dimension must be contiguous")
    for s in t.stride()[:-1]:
        _need(s % align_elems == 0, f"{name}: strides must be multiples of {align_elems} elements")
    _need(t.data_ptr() % (2 * align_elems if t.dtype == torch.bfloat16 else 4 * align_elems) == 0,
          f"{name}: base pointer misaligned")


def _contig(t: torch.Tensor, name: str, dtype: torch.dtype) -> None:
    _need(t.dtype == dtype, f"{name}: expected {dtype}, got {t.dtype}")
    _need(t.is_contiguous(), f"{name}: must be contiguous")


# ================================================================== OpenAttention.flash
def flash_decode(q, k, v, sel_idx, exp_idx, kbar, vbar, log_n, *, proxy_per_kv: bool,
                 sm_scale: float, n_bins: int | None = None, n_split: int | None = None,
                 out: torch.Tensor | None = None, noalloc: bool = False) -> torch.Tensor:
    """Shared body of ours_flash / decode_expand_attention.  noalloc=True calls
    oa_flash_decode_noalloc (split partials in the library's fixed device array; nothing is
    allocated, so `out` must be given)."""
    dev = _dev(q, k, v, sel_idx, exp_idx, kbar, vbar, log_n)
    R, D = q.shape
    _need(D == HEAD_DIM, f"head_dim must be {HEAD_DIM}")
    _need(q.dtype == torch.bfloat16 and k.dtype == torch.bfloat16 and v.dtype == torch.bfloat16,
          "q, k, v must be bfloat16")
    _need(k.dim() == 3 and k.shape == v.shape and k.stride() == v.stride() and k.shape[2] == D,
          "k, v must be (B*HKV, Lmax, D) with identical strides")
    BH = k.shape[0]
    _need(R % BH == 0, "rows of q must be a multiple of the KV rows of k")
    _rows_contig(q, "q", 8)
    _rows_contig(k, "k", 8)
    _rows_contig(v, "v", 8)
    _need(sel_idx.dtype == torch.int32 and exp_idx.dtype == torch.int32, "indices must be int32")
    _need(sel_idx.shape[0] == R and exp_idx.shape[0] == R, "index rows must match q")
    _need(sel_idx.stride(-1) == 1 and exp_idx.stride(-1) == 1, "index rows must be contiguous")
    NB = kbar.shape[1] if n_bins is None else int(n_bins)
    _need(0 <= NB <= kbar.shape[1], "nb out of range")
    _need(kbar.shape == vbar.shape and kbar.stride() == vbar.stride() and kbar.dtype == vbar.dtype,
          "kbar and vbar must match")
    _need(kbar.dtype in (torch.bfloat16, torch.float32), "kbar/vbar must be bf16 or fp32")
    _need(kbar.shape[0] == (BH if proxy_per_kv else R) and kbar.shape[2] == D, "kbar shape")
    _rows_contig(kbar, "kbar", 8 if kbar.dtype == torch.bfloat16 else 4)
    _need(log_n.dtype == torch.float32 and log_n.shape[0] == R and log_n.stride(-1) == 1,
          "log_n must be fp32 (R, C)")
    _need(not noalloc or out is not None, "noalloc needs a caller-provided out")
    if out is None:
        out = torch.empty_like(q)
    _need(out.shape == q.shape and out.dtype in (torch.bfloat16, torch.float32) and out.stride(1) == 1,
          "out must be (R, 128) bf16 or fp32 with contiguous rows")
    out_f32 = 1 if out.dtype == torch.float32 else 0
    T = sel_idx.shape[1] + exp_idx.shape[1] + NB
    if n_split is None:
        # few rows cannot fill the GPU: split each row's list (reference: ours_graph.py:276)
        n_split = 1 if R >= 512 else max(2, min(16, (4096 // max(R, 1)), -(-T // 32)))
    n_split = max(1, int(n_split))
    if noalloc:
        lib.call("oa_flash_decode_noalloc",
                 _ptr(q), q.stride(0), _ptr(k), _ptr(v), k.stride(0), k.stride(1),
                 _ptr(sel_idx), sel_idx.stride(0), sel_idx.shape[1],
                 _ptr(exp_idx), exp_idx.stride(0), exp_idx.shape[1],
                 _ptr(kbar), _ptr(vbar), kbar.stride(0), kbar.stride(1),
                 1 if kbar.dtype == torch.float32 else 0, 1 if proxy_per_kv else 0,
                 _ptr(log_n), log_n.stride(0), NB, _ptr(out), out.stride(0), out_f32,
                 R, BH, D, float(sm_scale), n_split, _stream(dev))
        return out
    ws = None
    if n_split > 1:
        ws = torch.empty(R * n_split * (HEAD_DIM + 2), device=dev, dtype=torch.float32)
        ws_m = ws[: R * n_split]
        ws_l = ws[R * n_split: 2 * R * n_split]
        ws_acc = ws[2 * R * n_split:]
    lib.call("oa_flash_decode",
             _ptr(q), q.stride(0), _ptr(k), _ptr(v), k.stride(0), k.stride(1),
             _ptr(sel_idx), sel_idx.stride(0), sel_idx.shape[1],
             _ptr(exp_idx), exp_idx.stride(0), exp_idx.shape[1],
             _ptr(kbar), _ptr(vbar), kbar.stride(0), kbar.stride(1),
             1 if kbar.dtype == torch.float32 else 0, 1 if proxy_per_kv else 0,
             _ptr(log_n), log_n.stride(0), NB, _ptr(out), out.stride(0), out_f32,
             R, BH, D, float(sm_scale), n_split,
             _ptr(ws_m) if ws is not None else None, _ptr(ws_l) if ws is not None else None,
             _ptr(ws_acc) if ws is not None else None, _stream(dev))
    return out


def ours_flash(q, k, v, sel_idx, exp_idx, kbar, vbar, log_n, nb=None):
    """q:(R,D) k,v:(B*HKV,Lmax,D) sel:(R,Ns) exp:(R,Ne) int32 (-1 = pad); kbar,vbar:(R,C,D);
    log_n:(R,C) natural log, -inf = no proxy.  nb overrides the proxy count (0 = P3 off).
    Same contract as inference/methods_eager.py:161-172; sm_scale = D**-0.5."""
    return flash_decode(q, k, v, sel_idx, exp_idx, kbar, vbar, log_n, proxy_per_kv=False,
                        sm_scale=HEAD_DIM ** -0.5, n_bins=nb)


def decode_expand_attention(q, k, v, sel_idx, exp_idx, kbar, vbar, log_n, sm_scale=None,
                            block_n=64, block_b=64, num_warps=4):
    """q:(BQ,D) k,v:(BH,K,D) sel_idx:(BQ,N_SEL) exp_idx:(BQ,N_EXP) kbar,vbar:(BH,NB,D)
    log_n:(BQ,NB) -> (BQ,D).  Same contract as triton_expand_decode.py:139-165; the Triton
    tuning arguments (block_n, block_b, num_warps) are accepted and ignored."""
    D = q.shape[1]
    scale = D ** -0.5 if sm_scale is None else float(sm_scale)
    return flash_decode(q, k, v, sel_idx, exp_idx, kbar, vbar, log_n, proxy_per_kv=True,
                        sm_scale=scale)


# ================================================================== decode-stage kernels
def index_update(K, V, st, n_dev: torch.Tensor, rmax: int) -> None:
    """The token at n-1 joins the index (ours_graph.py:43-90).  st: LayerState-like object
    with codes, U, scale, W, colmean, cent, asg, nb, Sk, Sk2, Sv, reclist, reccnt (one layer,
    all batch rows, flattened to rows)."""
    dev = _dev(K, V, n_dev)
    BH, Lmax, D = K.shape
    R = st.nb.shape[0]
    C = st.nb.shape[1]
    lib.call("oa_index_update", _ptr(K), _ptr(V), K.stride(0), K.stride(1), R, BH, D,
             _ptr(st.codes), st.codes.shape[1], RANK_Q, _ptr(st.U), _ptr(st.scale), _ptr(st.W),
             _ptr(st.colmean), RANK_C, _ptr(st.cent), C, _ptr(st.asg), st.asg.stride(0),
             _ptr(st.asg8), st.asg8.stride(0), _ptr(st.nb), _ptr(st.Sk), _ptr(st.Sk2), _ptr(st.Sv), _ptr(st.reclist),
             _ptr(st.reccnt), rmax, _ptr(n_dev), _stream(dev))


def index_downdate(K, V, st, n_dev: torch.Tensor) -> None:
    """The token at n-1 leaves the cluster statistics (nb, Sk, Sk2, Sv) of every query row: the
    statistics step of index_update undone, so that a causal row ending before it sees the
    statistics of the keys it attends (multibin.py:2210-2218)."""
    dev = _dev(K, V, n_dev)
    BH, Lmax, D = K.shape
    R = st.nb.shape[0]
    C = st.nb.shape[1]
    _chk(K, "K", torch.bfloat16, (BH, Lmax, HEAD_DIM))
    _need(V.shape == K.shape and V.stride() == K.stride() and V.dtype == K.dtype, "V must match K")
    _chk(st.asg, "asg", torch.int32, (R, -Lmax))
    _chk(st.nb, "nb", torch.float32, (R, C), contiguous=True)
    _stats(R, C, (st.Sk, "Sk"), (st.Sk2, "Sk2"), (st.Sv, "Sv"))
    _chk(n_dev, "n_dev", torch.int32)
    lib.call("oa_index_downdate", _ptr(K), _ptr(V), K.stride(0), K.stride(1), R, BH, D, _ptr(st.asg),
             st.asg.stride(0), _ptr(st.nb), _ptr(st.Sk), _ptr(st.Sk2), _ptr(st.Sv), C, _ptr(n_dev),
             _stream(dev))


def index_prep(K, V, st, n_dev: torch.Tensor, rmax: int, q, limbs, fexp) -> None:
    """index_update and qgs_prep in one launch (same results as the two calls)."""
    dev = _dev(K, V, n_dev, q, limbs, fexp)
    BH, Lmax, D = K.shape
    R = st.nb.shape[0]
    C = st.nb.shape[1]
    _chk(K, "K", torch.bfloat16, (BH, Lmax, HEAD_DIM))
    _need(V.shape == K.shape and V.stride() == K.stride() and V.dtype == K.dtype, "V must match K")
    _chk(st.codes, "codes", torch.int8, (BH, -Lmax, RANK_Q), contiguous=True)
    _chk(st.asg, "asg", torch.int32, (R, -Lmax))
    _chk(st.asg8, "asg8", torch.uint8, (R, -Lmax))
    _chk(st.nb, "nb", torch.float32, (R, C), contiguous=True)
    _stats(R, C, (st.Sk, "Sk"), (st.Sk2, "Sk2"), (st.Sv, "Sv"))
    _chk(q, "q", torch.bfloat16, (R, HEAD_DIM))
    _chk(n_dev, "n_dev", torch.int32)
    _chk(limbs, "limbs", torch.int8, (BH, 16, RANK_Q), contiguous=True)
    _chk(fexp, "fexp", torch.int32, (R,), contiguous=True)
    _rows_contig(q, "q")
    lib.call("oa_index_prep", _ptr(K), _ptr(V), K.stride(0), K.stride(1), R, BH, D,
             _ptr(st.codes), st.codes.shape[1], RANK_Q, _ptr(st.U), _ptr(st.scale), _ptr(st.W),
             _ptr(st.colmean), RANK_C, _ptr(st.cent), C, _ptr(st.asg), st.asg.stride(0),
             _ptr(st.asg8), st.asg8.stride(0), _ptr(st.nb), _ptr(st.Sk), _ptr(st.Sk2), _ptr(st.Sv),
             _ptr(st.reclist), _ptr(st.reccnt), rmax, _ptr(n_dev), _ptr(q), q.stride(0),
             _ptr(limbs), _ptr(fexp), _stream(dev))


def qgs_prep(q, U, scale, limbs, fexp, zq_out=None) -> None:
    dev = _dev(q, U, scale, limbs, fexp)
    R = q.shape[0]
    BH = U.shape[0]
    _rows_contig(q, "q")
    lib.call("oa_qgs_prep", _ptr(q), q.stride(0), _ptr(U), _ptr(scale), R, BH, q.shape[1], RANK_Q,
             _ptr(limbs), _ptr(fexp), _ptr(zq_out), _stream(dev))


def qgs_scan(codes, limbs, fexp, S, TM, n_dev, ns: int, nl: int) -> None:
    dev = _dev(codes, limbs, fexp, S, TM, n_dev)
    BH, Lmax, rq = codes.shape
    lib.call("oa_qgs_scan", _ptr(codes), BH, Lmax, rq, _ptr(limbs), _ptr(fexp), _ptr(S), S.stride(0),
             _ptr(TM), TM.stride(0), _ptr(n_dev), ns, nl, _stream(dev))


def topk_select(S, TM, sel, n_dev, ns: int, nl: int, k_top: int) -> None:
    dev = _dev(S, TM, sel, n_dev)
    R = S.shape[0]
    lib.call("oa_topk_select", _ptr(S), S.stride(0), _ptr(TM), TM.stride(0), R, TM.shape[1],
             _ptr(sel), sel.stride(0), _ptr(n_dev), ns, nl, k_top, _stream(dev))


def qgs_scan_heads(codes, limbs, fexp, H, TM, n_dev, ns: int, nl: int, TMn=None) -> None:
    """The scan writing 16-bit key heads of the scores (int16 tensor H, raw bits) instead of
    fp32 scores; TM (exact tile maxima) as oa_qgs_scan; TMn (optional, like TM): each tile's
    least finite score (+inf without one), the range topq_heads bins with."""
    dev = _dev(codes, limbs, fexp, H, TM, n_dev)
    if H.dtype != torch.int16:
        raise ValueError("H must be int16 (16-bit key heads)")
    BH, Lmax, rq = codes.shape
    _chk(codes, "codes", torch.int8, (BH, Lmax, RANK_Q), contiguous=True)
    _chk(H, "H", torch.int16, (GROUP * BH, -Lmax))
    _chk(TM, "TM", torch.float32, (GROUP * BH, None))
    _tile_min(TM, TMn)
    _chk(limbs, "limbs", torch.int8, (BH, 16, RANK_Q), contiguous=True)
    _chk(fexp, "fexp", torch.int32, (GROUP * BH,), contiguous=True)
    _chk(n_dev, "n_dev", torch.int32)
    lib.call("oa_qgs_scan_heads", _ptr(codes), BH, Lmax, rq, _ptr(limbs), _ptr(fexp), _ptr(H),
             H.stride(0), _ptr(TM), TM.stride(0), _ptr(TMn), _ptr(n_dev), ns, nl, _stream(dev))


def _tile_min(TM, TMn) -> None:
    """TMn, when given, is laid out as TM (same shape and row stride)."""
    if TMn is not None and (TMn.dtype != torch.float32 or TMn.shape != TM.shape
                            or TMn.stride() != TM.stride() or TMn.device != TM.device):
        raise ValueError("TMn must be a float32 tensor with TM's shape, strides and device")


def topk_select_heads(H, TM, sel, n_dev, ns: int, nl: int, k_top: int, codes, limbs, fexp) -> None:
    """Top-k over key-head rows: candidate scores recomputed exactly from the codes; the
    selected tokens' heads are set to that of -inf."""
    dev = _dev(H, TM, sel, n_dev, codes, limbs, fexp)
    R = H.shape[0]
    BH, Lmax, _ = codes.shape
    lib.call("oa_topk_select_heads", _ptr(H), H.stride(0), _ptr(TM), TM.stride(0), R, TM.shape[1],
             _ptr(sel), sel.stride(0), _ptr(n_dev), ns, nl, k_top, _ptr(codes), BH, Lmax,
             _ptr(limbs), _ptr(fexp), _stream(dev))


def errorgate(q, K, asg, sel, Sk, Sk2, nb, score, n_t, sm_scale: float) -> None:
    """wl1 cluster scores; sm_scale is the Python (double) scale, whose square is formed in
    double and rounded once, as the estimator does (multibin.py:643)."""
    dev = _dev(q, K, asg, sel, Sk, Sk2, nb, score, n_t)
    R, C = nb.shape
    BH = K.shape[0]
    lib.call("oa_errorgate", _ptr(q), q.stride(0), _ptr(K), K.stride(0), K.stride(1), R, BH,
             q.shape[1], _ptr(asg), asg.stride(0), _ptr(sel), sel.stride(0), sel.shape[1],
             _ptr(Sk), _ptr(Sk2), _ptr(nb), C, float(sm_scale), float(sm_scale) * float(sm_scale),
             _ptr(score), _ptr(n_t), _stream(dev))


def gate_fill(q, K, asg, sel, Sk, Sk2, nb, score, n_t, quota, sm_scale: float, E: int,
              qsk=None) -> None:
    """ErrorGate + water-filling (same results as errorgate then waterfill); qsk (R, C) fp32,
    when given, receives q . Sk of every cluster for residual_flash."""
    dev = _dev(q, K, asg, sel, Sk, Sk2, nb, score, n_t, quota)
    R, C = nb.shape
    BH = K.shape[0]
    _chk(q, "q", torch.bfloat16, (R, HEAD_DIM))
    _chk(K, "K", torch.bfloat16, (BH, None, HEAD_DIM))
    _chk(asg, "asg", torch.int32, (R, None))
    _chk(sel, "sel", torch.int32, (R, None))
    _stats(R, C, (Sk, "Sk"), (Sk2, "Sk2"))
    for t, name in ((nb, "nb"), (score, "score"), (n_t, "n_t"), (quota, "quota")):
        _chk(t, name, torch.float32, (R, C), contiguous=True)
    if qsk is not None and (qsk.shape != (R, C) or qsk.dtype != torch.float32 or not qsk.is_contiguous()):
        raise ValueError("qsk must be a contiguous (rows, C) float32 tensor")
    lib.call("oa_gate_fill", _ptr(q), q.stride(0), _ptr(K), K.stride(0), K.stride(1), R, BH,
             q.shape[1], _ptr(asg), asg.stride(0), _ptr(sel), sel.stride(0), sel.shape[1],
             _ptr(Sk), _ptr(Sk2), _ptr(nb), C, float(sm_scale), float(sm_scale) * float(sm_scale),
             int(E), _ptr(score), _ptr(n_t), _ptr(quota), _ptr(qsk), _stream(dev))


def topk_gate_fill(H, TM, n_dev, ns: int, nl: int, k_top: int, codes, limbs, fexp, q, K, asg, sel,
                   Sk, Sk2, nb, score, n_t, quota, sm_scale: float, E: int, qsk=None) -> None:
    """topk_select_heads then gate_fill (the same sel, marked heads, score, n_t, quota, qsk); one
    launch when the row fits the register top-k (its pooled ErrorGate computed while the top-k
    runs, then the selected tokens' correction and the fill).  sel has ns + nl + k_top columns."""
    dev = _dev(H, TM, n_dev, codes, limbs, fexp, q, K, asg, sel, Sk, Sk2, nb, score, n_t, quota)
    R, C = nb.shape
    BH, Lmax, _ = codes.shape
    _chk(H, "H", torch.int16, (R, -Lmax))
    _chk(TM, "TM", torch.float32, (R, None))
    _chk(codes, "codes", torch.int8, (BH, Lmax, RANK_Q), contiguous=True)
    _chk(limbs, "limbs", torch.int8, (BH, 16, RANK_Q), contiguous=True)
    _chk(fexp, "fexp", torch.int32, (R,), contiguous=True)
    _chk(q, "q", torch.bfloat16, (R, HEAD_DIM))
    _chk(K, "K", torch.bfloat16, (K.shape[0], None, HEAD_DIM))
    _chk(asg, "asg", torch.int32, (R, None))
    _chk(sel, "sel", torch.int32, (R, ns + nl + k_top))
    _stats(R, C, (Sk, "Sk"), (Sk2, "Sk2"))
    for t, name in ((nb, "nb"), (score, "score"), (n_t, "n_t"), (quota, "quota")):
        _chk(t, name, torch.float32, (R, C), contiguous=True)
    if qsk is not None and (qsk.shape != (R, C) or qsk.dtype != torch.float32 or not qsk.is_contiguous()):
        raise ValueError("qsk must be a contiguous (rows, C) float32 tensor")
    lib.call("oa_topk_gate_fill", _ptr(H), H.stride(0), _ptr(TM), TM.stride(0), TM.shape[1],
             _ptr(n_dev), ns, nl, k_top, _ptr(codes), Lmax, _ptr(limbs), _ptr(fexp), _ptr(q),
             q.stride(0), _ptr(K), K.stride(0), K.stride(1), R, K.shape[0], q.shape[1], _ptr(asg),
             asg.stride(0), _ptr(sel), sel.stride(0), _ptr(Sk), _ptr(Sk2), _ptr(nb), C,
             float(sm_scale), float(sm_scale) * float(sm_scale), int(E), _ptr(score), _ptr(n_t),
             _ptr(quota), _ptr(qsk), _stream(dev))


def qgs_scan_gate(codes, limbs, fexp, H, TM, n_dev, ns: int, nl: int, q, Sk, Sk2, nb, score, n_t,
                  sm_scale: float, qsk=None, TMn=None) -> None:
    """qgs_scan_heads and the pooled part of the ErrorGate in one launch: score, n_t (rows, C)
    of every cluster as if it held no selected token, and q . Sk_c into qsk."""
    dev = _dev(codes, limbs, fexp, H, TM, n_dev, q, Sk, Sk2, nb, score, n_t)
    BH, Lmax, rq = codes.shape
    R, C = nb.shape
    _chk(codes, "codes", torch.int8, (BH, Lmax, RANK_Q), contiguous=True)
    _chk(H, "H", torch.int16, (GROUP * BH, -Lmax))
    _chk(TM, "TM", torch.float32, (GROUP * BH, None))
    _tile_min(TM, TMn)
    _chk(limbs, "limbs", torch.int8, (BH, 16, RANK_Q), contiguous=True)
    _chk(fexp, "fexp", torch.int32, (GROUP * BH,), contiguous=True)
    _chk(n_dev, "n_dev", torch.int32)
    _chk(q, "q", torch.bfloat16, (R, HEAD_DIM))
    _need(R == GROUP * BH, "nb must have one row per query-head row")
    _stats(R, C, (Sk, "Sk"), (Sk2, "Sk2"))
    for t, name in ((nb, "nb"), (score, "score"), (n_t, "n_t")):
        _chk(t, name, torch.float32, (R, C), contiguous=True)
    if qsk is not None and (qsk.shape != (R, C) or qsk.dtype != torch.float32 or not qsk.is_contiguous()):
        raise ValueError("qsk must be a contiguous (rows, C) float32 tensor")
    lib.call("oa_qgs_scan_gate", _ptr(codes), BH, Lmax, rq, _ptr(limbs), _ptr(fexp), _ptr(H), H.stride(0),
             _ptr(TM), TM.stride(0), _ptr(TMn), _ptr(n_dev), ns, nl, _ptr(q), q.stride(0), _ptr(Sk), _ptr(Sk2), _ptr(nb),
             C, float(sm_scale), float(sm_scale) * float(sm_scale), _ptr(score), _ptr(n_t), _ptr(qsk),
             _stream(dev))


def topk_fix_fill(H, TM, n_dev, ns: int, nl: int, k_top: int, codes, limbs, fexp, q, K, asg, sel, Sk,
                  Sk2, nb, score, n_t, quota, sm_scale: float, E: int) -> None:
    """After qgs_scan_gate: the top-k over the heads, the ErrorGate of the clusters holding a
    selected token done again (score, n_t updated in place), the water-fill.  The same sel,
    marked heads, score, n_t and quota as topk_select_heads followed by gate_fill."""
    dev = _dev(H, TM, n_dev, codes, limbs, fexp, q, K, asg, sel, Sk, Sk2, nb, score, n_t, quota)
    R, C = nb.shape
    BH, Lmax, _ = codes.shape
    _chk(H, "H", torch.int16, (R, -Lmax))
    _chk(TM, "TM", torch.float32, (R, None))
    _chk(codes, "codes", torch.int8, (BH, Lmax, RANK_Q), contiguous=True)
    _chk(limbs, "limbs", torch.int8, (BH, 16, RANK_Q), contiguous=True)
    _chk(fexp, "fexp", torch.int32, (R,), contiguous=True)
    _chk(q, "q", torch.bfloat16, (R, HEAD_DIM))
    _chk(K, "K", torch.bfloat16, (K.shape[0], None, HEAD_DIM))
    _chk(asg, "asg", torch.int32, (R, None))
    _chk(sel, "sel", torch.int32, (R, ns + nl + k_top))
    _stats(R, C, (Sk, "Sk"), (Sk2, "Sk2"))
    for t, name in ((nb, "nb"), (score, "score"), (n_t, "n_t"), (quota, "quota")):
        _chk(t, name, torch.float32, (R, C), contiguous=True)
    lib.call("oa_topk_fix_fill", _ptr(H), H.stride(0), _ptr(TM), TM.stride(0), TM.shape[1],
             _ptr(n_dev), ns, nl, k_top, _ptr(codes), Lmax, _ptr(limbs), _ptr(fexp), _ptr(q),
             q.stride(0), _ptr(K), K.stride(0), K.stride(1), R, K.shape[0], q.shape[1], _ptr(asg),
             asg.stride(0), _ptr(sel), sel.stride(0), _ptr(Sk), _ptr(Sk2), _ptr(nb), C,
             float(sm_scale), float(sm_scale) * float(sm_scale), int(E), _ptr(score), _ptr(n_t),
             _ptr(quota), _stream(dev))


_ROW_MAPS: tuple = (("score", torch.float32), ("n_t", torch.float32), ("quota", torch.float32),
                    ("qsk", torch.float32))


def step(K, V, st, n_dev, q, w, sel, out, ns: int, nl: int, k_top: int, sm_scale: float, E: int, rmax: int,
         update: bool = True, qshift: int = 0, later: int = 0, stats=None) -> None:
    """The decode stages in one call (oa_step): index_prep (update) or qgs_prep, qgs_scan_heads,
    topk_gate_fill, topq_heads, residual_flash over the index st and the work buffers of w (limbs,
    fexp, H, TM, TMn, S, score, n_t, quota, qsk, exp_idx); the same outputs.  qshift > 0 or later > 0
    (update False): 2^qshift question rows per sequence, rows laid out ((kv << qshift) + i) * 4 + head
    in q, sel, out and w; stats = (nb, Sk, Sk2, Sv) receives their statistics."""
    dev = _dev(K)
    _on(dev, V, n_dev, q, w.limbs, w.fexp, w.H, w.TM, w.TMn, w.S, w.score, w.n_t, w.quota, w.qsk, w.exp_idx, sel, out,
        st.codes, st.asg, st.asg8, st.nb, st.Sk, st.Sk2, st.Sv, st.U, st.scale)
    if update:
        _on(dev, st.W, st.colmean, st.cent, st.reclist, st.reccnt)
    if stats is not None:
        _on(dev, *stats)
    BH, Lk, _ = K.shape
    Lmax = st.codes.shape[1]
    R, C = st.nb.shape
    Rv = R << qshift
    _chk(K, "K", torch.bfloat16, (BH, None, HEAD_DIM))
    _need(V.shape == K.shape and V.stride() == K.stride() and V.dtype == K.dtype, "V must match K")
    _need(R == GROUP * BH, "nb must have one row per query-head row")
    _chk(st.codes, "codes", torch.int8, (BH, None, RANK_Q), contiguous=True)
    # (the update writes ids, and question rows read them, at positions of K; a row without either reads
    # those of its own keys, which an index shorter than the cache may hold)
    _chk(st.asg, "asg", torch.int32, (R, -Lk if update or qshift or later else None))
    _chk(st.asg8, "asg8", torch.uint8, (R, -(max(Lk, Lmax) if update else Lmax)))
    _chk(st.nb, "nb", torch.float32, (R, C), contiguous=True)
    _stats(R, C, (st.Sk, "Sk"), (st.Sk2, "Sk2"), (st.Sv, "Sv"))
    if update:
        _need(Lmax >= Lk, "codes: fewer positions than K")
    _chk(n_dev, "n_dev", torch.int32)
    _chk(q, "q", torch.bfloat16, (Rv, HEAD_DIM))
    _chk(w.limbs, "limbs", torch.int8, (BH << qshift, 16, RANK_Q), contiguous=True)
    _chk(w.fexp, "fexp", torch.int32, (Rv,), contiguous=True)
    _chk(w.H, "H", torch.int16, (Rv, -Lmax))
    _chk(w.TM, "TM", torch.float32, (Rv, -((Lmax + 63) // 64)))
    _tile_min(w.TM, w.TMn)
    _chk(w.S, "S32", torch.float32, (Rv, -Lmax))
    _chk(sel, "sel", torch.int32, (Rv, ns + nl + k_top), contiguous=True)
    for name, dtype in _ROW_MAPS:
        _chk(getattr(w, name), name, dtype, (Rv, C), contiguous=True)
    _chk(w.exp_idx, "exp_idx", torch.int32, (Rv, None), contiguous=True)
    Ex = w.exp_idx.shape[1]
    _need(out.shape == (Rv, HEAD_DIM) and out.dtype in (torch.bfloat16, torch.float32) and out.stride(1) == 1,
          "out must be (rows, 128) bf16 or fp32 with contiguous rows")
    rs = (None,) * 4
    if qshift or later:
        _need(stats is not None, "question rows need their statistics' buffers")
        _chk(stats[0], "row nb", torch.float32, (Rv, C), contiguous=True)
        _stats(Rv, C, (stats[1], "row Sk"), (stats[2], "row Sk2"), (stats[3], "row Sv"))
        rs = tuple(t.data_ptr() for t in stats)
    a = lib.StepArgs(
        q.data_ptr(), q.stride(0), K.data_ptr(), V.data_ptr(), K.stride(0), K.stride(1), Rv, BH, HEAD_DIM,
        int(update), qshift, later, st.codes.data_ptr(), Lmax, st.U.data_ptr(), st.scale.data_ptr(),
        st.W.data_ptr(), st.colmean.data_ptr(), st.cent.data_ptr(), C, st.asg.data_ptr(), st.asg.stride(0),
        st.asg8.data_ptr(), st.asg8.stride(0), st.nb.data_ptr(), st.Sk.data_ptr(), st.Sk2.data_ptr(),
        st.Sv.data_ptr(), st.reclist.data_ptr(), st.reccnt.data_ptr(), rmax, w.limbs.data_ptr(),
        w.fexp.data_ptr(), w.H.data_ptr(), w.H.stride(0), w.TM.data_ptr(), w.TM.stride(0), w.TM.shape[1],
        _ptr(w.TMn), w.S.data_ptr(), w.S.stride(0), sel.data_ptr(), sel.stride(0), w.score.data_ptr(),
        w.n_t.data_ptr(), w.quota.data_ptr(), w.qsk.data_ptr(), w.exp_idx.data_ptr(), Ex, int(E), out.data_ptr(),
        out.stride(0), int(out.dtype == torch.float32), n_dev.data_ptr(), ns, nl, k_top, sm_scale,
        sm_scale * sm_scale, *rs)
    lib.call("oa_step", a, _stream(dev))


def waterfill(score, n_t, quota, E: int) -> None:
    dev = _dev(score, n_t, quota)
    R, C = score.shape
    lib.call("oa_waterfill", _ptr(score), _ptr(n_t), R, C, int(E), _ptr(quota), _stream(dev))


def topq(S, asg8, quota, exp_idx, n_dev, path: int | None = None) -> None:
    """Within-cluster top-q (exp_idx segments grouped by cluster, position order inside).
    path None: oa_topq; 0 / 1 / 2: oa_topq_path (both kernels / key-prefix only / linear-bin only,
    a row left to the key-prefix kernel then holding -2 in exp_idx[row, 0])."""
    dev = _dev(S, asg8, quota, exp_idx, n_dev)
    R, C = quota.shape
    Lmax = asg8.shape[1]
    E = exp_idx.shape[1]
    if path is None:
        lib.call("oa_topq", _ptr(S), S.stride(0), _ptr(asg8), asg8.stride(0), _ptr(quota), R, C,
                 Lmax, _ptr(exp_idx), E, _ptr(n_dev), _stream(dev))
    else:
        lib.call("oa_topq_path", _ptr(S), S.stride(0), _ptr(asg8), asg8.stride(0), _ptr(quota), R,
                 C, Lmax, _ptr(exp_idx), E, _ptr(n_dev), int(path), _stream(dev))


def topq_heads(H, asg8, quota, exp_idx, n_dev, codes, limbs, fexp, S32, path: int = 0, TM=None,
               TMn=None) -> None:
    """Within-cluster top-q over key-head rows (oa_topq_heads); S32 (fp32, rows as H) receives
    the exact scores of rows left to the key-prefix kernel.  path 2: the linear-bin kernel
    alone; path 3: every row through the key-prefix kernel.  TM, TMn (both or neither): the
    scan's tile maxima and minima, the row range taken from them (same result)."""
    dev = _dev(H, asg8, quota, exp_idx, n_dev, codes, limbs, fexp, S32)
    R, C = quota.shape
    Lmax = codes.shape[1]
    E = exp_idx.shape[1]
    _chk(H, "H", torch.int16, (R, -Lmax))
    _chk(asg8, "asg8", torch.uint8, (R, -Lmax))
    _chk(quota, "quota", torch.float32, (R, C), contiguous=True)
    _chk(exp_idx, "exp_idx", torch.int32, (R, E), contiguous=True)
    _chk(codes, "codes", torch.int8, (R // GROUP, Lmax, RANK_Q), contiguous=True)
    _chk(limbs, "limbs", torch.int8, (R // GROUP, 16, RANK_Q), contiguous=True)
    _chk(fexp, "fexp", torch.int32, (R,), contiguous=True)
    _chk(S32, "S32", torch.float32, (R, -Lmax))
    if (TM is None) != (TMn is None):
        raise ValueError("TM and TMn are given together")
    if TM is not None:
        _chk(TM, "TM", torch.float32, (R, -((Lmax + 63) // 64)))
        _tile_min(TM, TMn)
    lib.call("oa_topq_heads", _ptr(H), H.stride(0), _ptr(asg8), asg8.stride(0), _ptr(quota), R, C,
             Lmax, _ptr(exp_idx), E, _ptr(n_dev), _ptr(codes), codes.shape[0], _ptr(limbs),
             _ptr(fexp), _ptr(S32), S32.stride(0), _ptr(TM), _ptr(TMn),
             TM.stride(0) if TM is not None else 0, int(path), _stream(dev))


def residual(K, V, asg, sel, exp_idx, quota, n_t, Sk, Sv, kbar_r, vbar_r, log_n) -> None:
    dev = _dev(K, V, asg, sel, exp_idx, quota, n_t, Sk, Sv, kbar_r, vbar_r, log_n)
    R, C = quota.shape
    BH = K.shape[0]
    lib.call("oa_residual", _ptr(K), _ptr(V), K.stride(0), K.stride(1), R, BH, K.shape[2],
             _ptr(asg), asg.stride(0), _ptr(sel), sel.stride(0), sel.shape[1], _ptr(exp_idx),
             exp_idx.shape[1], _ptr(quota), _ptr(n_t), _ptr(Sk), _ptr(Sv), C, _ptr(kbar_r),
             _ptr(vbar_r), _ptr(log_n), _stream(dev))


def residual_flash(q, K, V, asg, sel, exp_idx, quota, n_t, Sk, Sv, out, sm_scale: float,
                   qsk=None) -> None:
    """Residual proxies + fused softmax; qsk (R, C) fp32 from gate_fill, when given, replaces the
    kernel's own pass over Sk (same quantity, summed in another order)."""
    dev = _dev(q, K, V, asg, sel, exp_idx, quota, n_t, Sk, Sv, out)
    R, C = quota.shape
    BH = K.shape[0]
    _chk(q, "q", torch.bfloat16, (R, HEAD_DIM))
    _chk(K, "K", torch.bfloat16, (BH, None, HEAD_DIM))
    _need(V.shape == K.shape and V.stride() == K.stride() and V.dtype == K.dtype, "V must match K")
    _chk(asg, "asg", torch.int32, (R, None))
    _chk(sel, "sel", torch.int32, (R, None))
    _chk(exp_idx, "exp_idx", torch.int32, (R, None), contiguous=True)
    for t, name in ((quota, "quota"), (n_t, "n_t")):
        _chk(t, name, torch.float32, (R, C), contiguous=True)
    _stats(R, C, (Sk, "Sk"), (Sv, "Sv"))
    if qsk is not None and (qsk.shape != (R, C) or qsk.dtype != torch.float32 or not qsk.is_contiguous()):
        raise ValueError("qsk must be a contiguous (rows, C) float32 tensor")
    _need(out.shape == (R, HEAD_DIM) and out.dtype in (torch.bfloat16, torch.float32) and out.stride(1) == 1,
          "out must be (R, 128) bf16 or fp32 with contiguous rows")
    lib.call("oa_residual_flash", _ptr(q), q.stride(0), _ptr(K), _ptr(V), K.stride(0), K.stride(1),
             R, BH, K.shape[2], _ptr(asg), asg.stride(0), _ptr(sel), sel.stride(0), sel.shape[1],
             _ptr(exp_idx), exp_idx.shape[1], _ptr(quota), _ptr(n_t), _ptr(Sk), _ptr(Sv), C,
             float(sm_scale), _ptr(out), out.stride(0), 1 if out.dtype == torch.float32 else 0,
             _ptr(qsk), _stream(dev))


# key chunks per KV row of the dense comparator: measured best both at B = 32 (8192 workgroups:
# 725 us against 980 with 256 chunks) and at B = 1 (54 us against 117: the combine walks every
# chunk)
DENSE_SPLITS = 32


def dense_decode(q, K, V, n_dev, out=None, sm_scale: float | None = None, nsplit: int | None = None,
                 ws: torch.Tensor | None = None) -> torch.Tensor:
    """Dense decode attention over [0, n) (graph_runner.py:259-312 comparator)."""
    dev = _dev(q, K, V, n_dev)
    R, D = q.shape
    BH, Lmax, _ = K.shape
    _rows_contig(q, "q", 8)
    _rows_contig(K, "K", 8)
    if nsplit is None:
        nsplit = DENSE_SPLITS
    if out is None:
        out = torch.empty_like(q)
    need = R * nsplit * (HEAD_DIM + 2)
    if ws is None or ws.numel() < need:
        ws = torch.empty(need, device=dev, dtype=torch.float32)
    scale = D ** -0.5 if sm_scale is None else sm_scale
    lib.call("oa_dense_decode", _ptr(q), q.stride(0), _ptr(K), _ptr(V), K.stride(0), K.stride(1), R,
             BH, D, Lmax, _ptr(n_dev), float(scale), nsplit, _ptr(ws[: R * nsplit]),
             _ptr(ws[R * nsplit: 2 * R * nsplit]), _ptr(ws[2 * R * nsplit: need]), _ptr(out),
             out.stride(0), _stream(dev))
    return out


def _watched() -> bool:
    """Whether something on this thread has to see a torch operation that is run now, which a library
    call would hide from it: a tracer, a dispatch or function mode (a default device is none), autocast
    to another type."""
    if (torch.jit.is_tracing() or torch.compiler.is_compiling() or torch._C._len_torch_dispatch_stack()
            or torch._ops._len_torch_dispatch_stack_pre_dispatch()
            or torch.is_autocast_enabled("cuda") and torch.get_autocast_dtype("cuda") != torch.bfloat16):
        return True
    return torch._C._len_torch_function_stack() > 0 and any(
        not isinstance(m, DeviceContext) for m in _get_current_function_mode_stack())


def prefill_attn_ok(q, k, v, sm_scale: float = 1.0) -> bool:
    """Whether prefill_attn takes these arguments: a scale that is not negative (the running maximum is
    taken before it is applied), plain bf16 tensors on the current HIP device, of Llama-3.1-8B's head
    layout, one sequence, rows of dims contiguous, 16-byte aligned, and nothing that would have to see
    the operation (autograd in either mode, a functional transform, what _watched names)."""
    if (sm_scale is None or not sm_scale >= 0 or _watched() or q.dim() != 4 or k.dim() != 4 or q.shape[0] != 1 or k.shape[0] != 1 or k.shape != v.shape
            or q.shape[3] != HEAD_DIM or k.shape[3] != HEAD_DIM or q.shape[1] != GROUP * k.shape[1]
            or q.shape[2] != k.shape[2] or not 1 <= q.shape[2] <= 1 << 24):
        return False
    for t in (q, k, v):
        if (type(t) not in (torch.Tensor, torch.nn.Parameter) or t.dtype != torch.bfloat16
                or t.device.type != "cuda" or t.device != q.device or t.is_neg() or t.stride(3) != 1
                or t.stride(1) % 8 or t.stride(2) % 8 or t.stride(2) < HEAD_DIM or t.stride(2) > 1 << 24
                or torch._C._functorch.is_functorch_wrapped_tensor(t) or t.data_ptr() % 16):
            return False
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return False
    return torch.autograd.forward_ad._current_level < 0 and q.device.index == torch.cuda.current_device()


def prefill_attn(q, k, v, sm_scale: float) -> torch.Tensor:
    """Dense causal attention of one prompt (oa_prefill_attn): q (1, HQ, T, 128), k, v (1, HKV, T, 128)
    bf16, any head and position strides that prefill_attn_ok admits -> (1, HQ, T, 128), a view of
    position-major rows."""
    dev = _dev(q, k, v)
    _need(prefill_attn_ok(q, k, v, sm_scale), "q, k, v: one sequence of bf16 rows of 128 aligned dims, "
          "HQ = 4 HKV, a scale >= 0")
    _, HQ, T, _ = q.shape
    out = torch.empty(1, T, HQ, HEAD_DIM, device=dev, dtype=torch.bfloat16)
    lib.call("oa_prefill_attn", _ptr(q), q.stride(1), q.stride(2), _ptr(k), k.stride(1), k.stride(2), _ptr(v),
             v.stride(1), v.stride(2), HQ, k.shape[1], T, HEAD_DIM, float(sm_scale), _ptr(out), out.stride(2),
             out.stride(1), _stream(dev))
    return out.transpose(1, 2)


# ================================================================== 4-bit paged cache
# An eager decode step calls these once per layer, and their checks were two thirds of a call's time on the
# host.  So what depends on sizes, strides and types alone (_*_sizes below) is looked up by those, and only
# what can differ between tensors of the same sizes is looked at in every call: devices, alignment, gradients.
# Numbers go in as Python's own, so that no tensor's value is taken for another's.
_DT = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
KV4_BLOCK = 32             # values that share a scale
_GRID = (1 << 24) - 1      # workgroups of 256 threads along a grid's axis, whose threads are counted in 32 bits
_raw_stream = torch._C._cuda_getCurrentRawStream
_get_device = torch._C._cuda_getDevice
_forward_ad = torch.autograd.forward_ad
_sizes = functools.lru_cache(maxsize=1024)


def _where(*ts) -> int:
    """The index of the device that all these tensors are on."""
    i = ts[0].get_device()
    for t in ts:
        if t is not None and t.get_device() != i or i < 0:
            _dev(*ts)
            raise RuntimeError(f"tensors on different devices: {[u.device for u in ts if u is not None]}")
    return i


def _run(i: int, name: str, *args) -> None:
    """lib.call on device i's current stream, with i the current device for the launch."""
    if i == _get_device():
        lib.call(name, *args, _raw_stream(i))
    else:
        with torch.cuda.device(i):
            lib.call(name, *args, _raw_stream(i))


def _plain(*ts) -> None:
    """Tensors whose data a kernel may take as it stands, with no gradient to be formed: these
    operators have no backward pass, and would cut a graph in silence."""
    grad, dual = torch.is_grad_enabled(), _forward_ad._current_level >= 0
    for t in ts:
        if t is not None:
            if grad and t.requires_grad:
                raise ValueError("a tensor requires a gradient, and this operator has no backward pass (call it under "
                                 "torch.no_grad())")
            if dual and _forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError("a tensor carries a forward-mode tangent, which this operator would drop")
            if t.is_neg():
                raise ValueError("a lazily negated view (call resolve_neg())")


def _aligned(p: int) -> None:
    """p: pointers or-ed together"""
    if p % 16:
        raise ValueError("rows, tables, weights and caches must start at multiples of 16 bytes")


def _m(t):
    return None if t is None else (t.shape, t.stride(), t.dtype)


def _row_strides(T: int, H: int, Dh: int, stride: tuple, dtype: torch.dtype, name: str, out: bool = False) -> tuple:
    """(token stride, head stride) of rows (T, H, Dh) that are loaded 16 bytes at a time; of an output, rows that
    do not overlap.  The stride of a single token or head, which is free, counts as 0."""
    s0, s1, s2 = stride
    if T <= 1:
        s0 = 0
    if H <= 1:
        s1 = 0
    if T * H:
        _need((s0 | s1) % (4 if dtype is torch.float32 else 8) == 0 and s2 == 1,
              f"{name}: contiguous rows that start at multiples of 16 bytes (strides {stride})")
        _need(not out or (H <= 1 or s1 >= Dh) and (T <= 1 or s0 >= s1 * (H - 1) + Dh)
              or (T <= 1 or s0 >= Dh) and (H <= 1 or s1 >= s0 * (T - 1) + Dh), f"{name}: rows overlap")
    return s0, s1


def _rows(T: int, H: int, stride: tuple, n: int, Dh: int) -> tuple:
    """Where rows of Dh values of n bytes lie from their first: (bytes to the last one's end, tokens, heads, bytes between
    tokens and between heads, bytes of a row)"""
    s0, s1 = stride
    return (n * ((T - 1) * s0 + (H - 1) * s1 + Dh) if T * H else 0), T, H, n * s0, n * s1, n * Dh


@_sizes
def _meet(d: int, a: tuple, b: tuple) -> bool:
    """Whether rows a (_rows), which do not overlap one another, share a byte with rows b that begin d bytes behind them.
    Equal strides, as of views of one product: whether d is a sum of strides and less than a row, exactly, whatever the
    sizes; others by the rows' sorted places."""
    _, Ta, Ha, a0, a1, wa = a
    _, Tb, Hb, b0, b1, wb = b
    if not ((a0 == b0 or Ta == 1 or Tb == 1) and (a1 == b1 or Ha == 1 or Hb == 1)):
        x, y = (np.add.outer(s0 * np.arange(T), s1 * np.arange(H)).ravel() for _, T, H, s0, s1, _ in (a, b))
        x.sort()
        y += d
        at = np.searchsorted(x, y - wa, side="right")       # the first of a's rows that ends behind one of b's
        return bool((x[np.minimum(at, x.size - 1)] < y + wb)[at < x.size].any())
    # d = i S + j s + e: steps i, j from a row of b to one of a, -wb < e < wa
    (S, lo, hi), (s, l, h) = sorted(((a0 if Ta > 1 else b0, 1 - Tb, Ta - 1), (a1 if Ha > 1 else b1, 1 - Hb, Ha - 1)), reverse=True)
    for i in range(max(lo, -((h * s + wa - 1 - d) // S)), min(hi, (d - l * s + wb - 1) // S) + 1) if S else (0,):
        x = d - i * S
        if (max(l, -((wa - 1 - x) // s)) <= min(h, (x + wb - 1) // s)) if s else -wb < x < wa:
            return True
    return False


def _apart(name: str, p: int, rows: tuple, *others) -> None:
    """An output's rows at p, which share no byte with the others (address, _rows)."""
    end = p + rows[0]
    for x, r in others:
        if x < end and p < x + r[0] and rows[0] and r[0] and _meet(x - p, rows, r):
            raise ValueError(f"{name}: its rows share memory with what the call reads, or writes besides")


def _int_vector(shape: tuple, stride: tuple, dtype: torch.dtype, n: int, name: str) -> None:
    _need(dtype is torch.int32 and shape == (n,) and (n <= 1 or stride[0] == 1),
          f"{name}: ({n},) int32, contiguous (got {tuple(shape)} {dtype})")


@_sizes
def _rope_sizes(qs, qst, dt, ks, kst, kt, ps, pst, pt, cs, cst, ct, ss, sst, st, wq, wk, eps, qo, ko) -> tuple:
    _need(len(qs) == 3 and len(ks) == 3 and dt in _DT and kt is dt, "q, k: (T, HQ, D) and (T, HKV, D), both bf16, fp16 or fp32")
    T, HQ, Dh = qs
    HKV = ks[1]
    _need(ks[0] == T and ks[2] == Dh and Dh in (64, 128, 256) and T * (HQ + HKV) <= 1 << 27,
          "q, k: the same tokens, heads of 64, 128 or 256, at most 2^27 rows")
    _need(pt in (torch.int32, torch.int64) and ps == (T,) and (T <= 1 or pst[0] == 1), f"pos: ({T},) int32 or int64, contiguous")
    f32 = torch.float32
    _need(len(cs) == 2 and cs[1] == Dh // 2 and cs[0] >= 1 and ss == cs and ct is f32 and st is f32 and cst == sst and cst[1] == 1
          and (cs[0] == 1 or cst[0] % 4 == 0), f"cos, sin: (positions, {Dh // 2}) fp32 rows of one stride, of whole 16 bytes")
    for w, name in ((wq, "wq"), (wk, "wk")):
        _need(w is None or w[0] == (Dh,) and w[1] == (1,) and w[2] is dt, f"{name}: ({Dh},) of q's type, contiguous")
    _need(eps >= 0, "eps: not negative")
    for o, s, name in ((qo, qs, "q_out"), (ko, ks, "k_out")):
        _need(o is None or o[0] == s and o[2] is dt, f"{name}: as {name[0]}")
    qst, kst = _row_strides(T, HQ, Dh, qst, dt, "q"), _row_strides(T, HKV, Dh, kst, dt, "k")
    qo = (HQ * Dh, Dh) if qo is None else _row_strides(T, HQ, Dh, qo[1], dt, "q_out", True)
    ko = (HKV * Dh, Dh) if ko is None else _row_strides(T, HKV, Dh, ko[1], dt, "k_out", True)
    n, table = dt.itemsize, (cst[0] if cs[0] > 1 else 0, cs[0])
    return (T, HQ, HKV, Dh, qst, kst, qo, ko, (T, HQ, HKV, Dh, _DT[dt]), pt is torch.int64, table,
            (_rows(T, HQ, qst, n, Dh), _rows(T, HKV, kst, n, Dh), _rows(T, HQ, qo, n, Dh), _rows(T, HKV, ko, n, Dh),
             _rows(1, 1, (0, 0), pt.itemsize, T), _rows(cs[0], 1, (table[0], 0), 4, Dh // 2), _rows(1, 1, (0, 0), n, Dh)))


def qk_norm_rope(q, k, pos, cos, sin, wq=None, wk=None, eps: float = 1e-6, q_out=None, k_out=None):
    """Query and key rows of a layer, each head normalised (x / sqrt(mean(x^2) + eps) * w) and turned to
    its token's position (halves of the head dimension as pairs) in one pass, fp32 inside.
    q (T, HQ, D), k (T, HKV, D) bf16, fp16 or fp32, D 64, 128 or 256, any token and head strides of whole
    16 bytes (views of one product, say); pos (T,) int32 or int64; cos, sin (P, D / 2) fp32; wq, wk (D,)
    of q's type, None for a rotation alone.  A token of negative position (padding) gives zeros, one of P
    or more NaN.  Returns (q_out, k_out), contiguous unless given; either may be its input, and shares no
    memory with the other tensors."""
    i = _where(q, k, pos, cos, sin, wq, wk, q_out, k_out)
    T, HQ, HKV, Dh, qst, kst, qo, ko, sizes, wide, table, lie = _rope_sizes(
        q.shape, q.stride(), q.dtype, k.shape, k.stride(), k.dtype, pos.shape, pos.stride(), pos.dtype, cos.shape, cos.stride(),
        cos.dtype, sin.shape, sin.stride(), sin.dtype, _m(wq), _m(wk), float(eps), _m(q_out), _m(k_out))
    _plain(q, k, cos, sin, wq, wk, q_out, k_out)
    given = (q_out is not None) + 2 * (k_out is not None)
    if q_out is None:
        q_out = q.new_empty(T, HQ, Dh)
    if k_out is None:
        k_out = k.new_empty(T, HKV, Dh)
    qp, kp, cp, sp, qop, kop = q.data_ptr(), k.data_ptr(), cos.data_ptr(), sin.data_ptr(), q_out.data_ptr(), k_out.data_ptr()
    wqp, wkp = _ptr(wq), _ptr(wk)
    if T:
        _aligned((qp | qop if HQ else 0) | (kp | kop if HKV else 0) | cp | sp | (wqp or 0) | (wkp or 0))
    if given:                              # each its own input, or apart from what is read and from each other
        lq, lk, lqo, lko, lp, lt, lw = lie
        rest = (pos.data_ptr(), lp), (cp, lt), (sp, lt), (wqp or 0, lw), (wkp or 0, lw)
        if given & 1:
            _apart("q_out", qop, lqo, (kp, lk), (kop, lko), *rest, *(() if qop == qp and qo == qst else ((qp, lq),)))
        if given & 2:
            _apart("k_out", kop, lko, (qp, lq), (qop, lqo), *rest, *(() if kop == kp and ko == kst else ((kp, lk),)))
    _run(i, "oa_qk_norm_rope", qp, *qst, kp, *kst, *sizes, pos.data_ptr(), wide, cp, sp, *table, wqp, wkp, eps, qop, *qo,
         kop, *ko)
    return q_out, k_out


def _page(page: int) -> None:
    _need(32 <= page <= 1024 and page & (page - 1) == 0, f"page: a power of two, 32 to 1024 (got {page})")


def _table_sizes(ts, tst, tt, page: int) -> tuple:
    """(row stride, rows, width) of a table of page ids"""
    _need(len(ts) == 2 and tt is torch.int32, "table: (requests, width) int32")
    B, width = ts
    _need(width >= 1 and width * page <= 1 << 30 and (width == 1 or tst[1] == 1) and (B <= 1 or tst[0] >= width) and B <= 1 << 24,
          "table: contiguous rows of at most 2^30 tokens, at most 2^24 requests")
    return max(tst[0], width), B, width


@_sizes
def _pages_sizes(page, ts, tst, tt, fs, fst, ft, count, lens, nfree, status, what) -> tuple:
    _page(page)
    stride, B, width = _table_sizes(ts, tst, tt, page)
    _need(len(fs) == 1, "free: (pages,) int32")
    NP = fs[0]
    _need(B >= 1 and NP >= 1 and NP * page < 1 << 31, "at least one request and page; a pool of fewer than 2^31 tokens")
    _int_vector(fs, fst, ft, NP, "free")
    for m, n, name in ((count, B, what), (lens, B, "lens"), (nfree, 1, "nfree"), (status, 1, "status")):
        _int_vector(*m, n, name)
    return stride, B, (B, width, NP, page)


def kv_pages_extend(add, lens, table, free, nfree, status, page: int, total: int):
    """Requests add tokens (add (B,) int32, lens (B,) what they hold): pages popped off the stack of free
    ids (free, height nfree (1,)) into their rows of table (B, width), lens grown.  Returns int32 (slots
    (total,), pos (total,), cu (B + 1,)): page id * page + offset and position of the new tokens, request
    after request, from cu[i] on; -1 behind cu[B].  All on the device, so that a captured step can cross
    into new pages.  For all requests or for none: where a count is negative, a request outgrows its row
    (status |= 1), free pages do not reach (2) or there are more than `total` new tokens (4), nothing
    changes, slots and pos are -1 and cu is 0; status (1,) is the caller's to look at and to clear."""
    i = _where(add, lens, table, free, nfree, status)
    stride, B, sizes = _pages_sizes(index(page), table.shape, table.stride(), table.dtype, free.shape, free.stride(), free.dtype,
                                    _m(add), _m(lens), _m(nfree), _m(status), "add")
    if not 0 <= total <= 1 << 30:
        raise ValueError("total: 0 to 2^30")
    slots, pos, cu = add.new_empty(total), add.new_empty(total), add.new_empty(B + 1)
    ws = add.new_empty(3 * B + 1) if B > 1024 or total > 2048 else None
    _run(i, "oa_kv_pages_extend", add.data_ptr(), lens.data_ptr(), table.data_ptr(), stride, free.data_ptr(), nfree.data_ptr(),
         status.data_ptr(), *sizes, total, slots.data_ptr(), pos.data_ptr(), cu.data_ptr(), _ptr(ws))
    return slots, pos, cu


def kv_pages_truncate(keep, lens, table, free, nfree, status, page: int) -> None:
    """Request i keeps its first min(keep[i], lens[i]) tokens (keep[i] < 0: all; 0: the request ends); pages
    it no longer needs go back to the stack and leave the table (-1).  A truncation to the lengths before
    an extension undoes it.  For all requests or for none: nothing changes where the stack would outgrow `free`
    (status |= 2) or a length lies outside of its row (1)."""
    i = _where(keep, lens, table, free, nfree, status)
    stride, B, sizes = _pages_sizes(index(page), table.shape, table.stride(), table.dtype, free.shape, free.stride(), free.dtype,
                                    _m(keep), _m(lens), _m(nfree), _m(status), "keep")
    ws = keep.new_empty(3 * B + 1) if B > 256 else None
    _run(i, "oa_kv_pages_truncate", keep.data_ptr(), lens.data_ptr(), table.data_ptr(), stride, free.data_ptr(),
         nfree.data_ptr(), status.data_ptr(), *sizes, _ptr(ws))


@_sizes
def _kv4_sizes(kcs, kst, kct, kss, sst, ksdt, vcs, vst, vct, vss, vsst, vsdt) -> tuple:
    """(page strides, pages, page) of a 4-bit cache's tensors, its heads and head dimension; pages may lie apart (a
    layer of a larger tensor)."""
    _need(len(kcs) == 4, "kc: (pages, heads, page, D / 2) uint8")
    NP, HKV, page, half = kcs
    blocks = half // (KV4_BLOCK // 2)
    _page(page)
    _need(half in (32, 64) and NP >= 1 and HKV >= 1 and NP * page < 1 << 31,
          f"cache: head dimension 64 or 128 (got {2 * half}), at least one page and head, fewer than 2^31 slots")
    u8 = torch.uint8
    _need(vcs == kcs and kss == (NP, HKV, page, blocks) and vss == kss and kct is u8 and ksdt is u8 and vct is u8 and vsdt is u8,
          f"cache: codes ({NP}, {HKV}, {page}, {half}), scales ({NP}, {HKV}, {page}, {blocks}), uint8")
    c0, s0 = (kst[0], sst[0]) if NP > 1 else (HKV * page * half, HKV * page * blocks)
    _need(vst == kst and vsst == sst and kst[1:] == (page * half, half, 1) and sst[1:] == (page * blocks, blocks, 1)
          and c0 >= HKV * page * half and s0 >= HKV * page * blocks and c0 < 1 << 32 and (c0 | s0) % 16 == 0,
          "cache: contiguous pages, those of k and v at one distance, of whole 16 bytes, under 2^32")
    return (c0, s0, NP, page), HKV, 2 * half


def _kv4_cache(kc, ks, vc, vs) -> tuple:
    """A 4-bit cache's pointers and sizes (_kv4_sizes)."""
    sizes = _kv4_sizes(kc.shape, kc.stride(), kc.dtype, ks.shape, ks.stride(), ks.dtype, vc.shape, vc.stride(), vc.dtype,
                       vs.shape, vs.stride(), vs.dtype)
    p = kc.data_ptr(), ks.data_ptr(), vc.data_ptr(), vs.data_ptr()
    _aligned(p[0] | p[1] | p[2] | p[3])
    return p, *sizes


@_sizes
def _write_sizes(HKV, Dh, ks, kst, kt, vs, vst, vt, ss, sst, st) -> tuple:
    _need(len(ks) == 3 and ks[1:] == (HKV, Dh) and vs == ks and kt in _DT and vt is kt and ks[0] * HKV <= 1 << 26,
          f"k, v: (T, {HKV}, {Dh}), both bf16, fp16 or fp32, at most 2^26 rows")
    T = ks[0]
    _int_vector(ss, sst, st, T, "slots")
    return _row_strides(T, HKV, Dh, kst, kt, "k"), _row_strides(T, HKV, Dh, vst, kt, "v"), (T, HKV, Dh, _DT[kt])


def kv4_write(k, v, slots, kc, ks, vc, vs) -> None:
    """Key and value rows (T, HKV, D) bf16, fp16 or fp32 rounded to 4 bits (blocks of 32 with a power-of-two
    scale) and put at slots (T,) int32 = page id * page + offset of the cache kc, vc (pages, HKV, page,
    D / 2), ks, vs (pages, HKV, page, D / 32) uint8.  Rows of a slot outside of the cache (-1) are passed
    over.  The slots of one call are distinct (one given twice ends with codes and scales of either row)."""
    i = _where(k, v, slots, kc, ks, vc, vs)
    ps, where, HKV, Dh = _kv4_cache(kc, ks, vc, vs)
    kst, vst, sizes = _write_sizes(HKV, Dh, k.shape, k.stride(), k.dtype, v.shape, v.stride(), v.dtype, slots.shape,
                                   slots.stride(), slots.dtype)
    _plain(k, v)
    kp, vp = k.data_ptr(), v.data_ptr()
    if sizes[0]:
        _aligned(kp | vp)
    _run(i, "oa_kv4_write", kp, *kst, vp, *vst, *sizes, slots.data_ptr(), *ps, *where)


def kv4_read(slots, kc, ks, vc, vs, dtype: torch.dtype = torch.bfloat16):
    """The values (k, v), each (T, HKV, D) bf16 (which holds them exactly) or fp32, at slots (T,) int32 of a
    4-bit cache; zeros for a slot outside of it."""
    i = _where(slots, kc, ks, vc, vs)
    ps, where, HKV, Dh = _kv4_cache(kc, ks, vc, vs)
    T = slots.shape[0] if slots.dim() == 1 else 0
    _int_vector(slots.shape, slots.stride(), slots.dtype, T, "slots")
    if dtype not in (torch.bfloat16, torch.float32) or T * HKV > 1 << 26:
        raise ValueError("dtype: bf16 or fp32; at most 2^26 rows")
    k = kc.new_empty(T, HKV, Dh, dtype=dtype)
    v = kc.new_empty(T, HKV, Dh, dtype=dtype)
    _run(i, "oa_kv4_read", slots.data_ptr(), *ps, *where, k.data_ptr(), HKV * Dh, Dh, v.data_ptr(), HKV * Dh, Dh, T, HKV, Dh,
         _DT[dtype])
    return k, v


def kv4_chunk(cap: int, units: int, rows: int) -> int:
    """Keys per workgroup of kv4_attn, for `units` (sequence, KV head, query tile) triples of up to `cap` keys and
    `rows` query rows: two workgroups to a compute unit, but pieces of at least 384 keys (their start and end
    cost as much as some 300).  Where the rows are few and reading keys is the work, at most an eighth of the
    longest sequence (or 1024), so that a batch does not wait for one piece of it: 61 sequences of 1 to
    16001 keys take 107 us whole, 58 in pieces of 4096, 44 of 2048, 45 of 1024 and 50 of 512 (captured)."""
    n = max(cap * units // 512, 384)
    if rows <= 64:
        n = max(min(n, max(cap // 8, 1024)), 384)
    return min(-(-n // 128), -(-cap // 128)) * 128


@_sizes
def _attn_sizes(HKV, Dh, where, qs, qst, qt, ts, tst, tt, ls, lst, lt, cu, max_q, sm_scale, max_len, o, rule) -> tuple:
    # rule: kv4_chunk, a part of what is looked up, so that no call gets the pieces of another rule
    c0, s0, NP, page = where
    tstride, B, width = _table_sizes(ts, tst, tt, page)
    _need(len(qs) == 3 and qs[2] == Dh and qt is torch.bfloat16 and qs[1] >= 1 and qs[1] % HKV == 0,
          f"q: (T, a multiple of {HKV}, {Dh}) bf16")
    T, HQ, _ = qs
    _int_vector(ls, lst, lt, B, "lens")
    if cu is not None:
        _int_vector(*cu, B + 1, "cu_q")
    else:
        _need(T == B and max_q == 1, "without cu_q every sequence has one row of q")
    scale = Dh ** -0.5 if sm_scale is None else sm_scale
    _need(1 <= max_q <= (1 << 30) // (HQ // HKV) and scale == scale and (max_len is None or max_len >= 0),
          "max_q: at least 1; sm_scale: not NaN; max_len: not negative")
    _need(o is None or o[0] == qs and o[2] is torch.bfloat16, "out: as q")
    rows = max_q * (HQ // HKV)
    cap = max(1, width * page if max_len is None else min(max_len, width * page))
    units = B * HKV * -(-rows // (8 if rows <= 8 else 16 if rows <= 16 else 32 if rows <= 64 else 128))
    # (the join's grid holds 65535 sequences; so many need no pieces to fill the card)
    chunk = rule(cap, units, rows) if B <= 65535 else -(-cap // 128) * 128
    nchunk = -(-cap // chunk)
    _need(units * nchunk <= _GRID and B * HKV * HKV < 1 << 32,
          f"at most {_GRID} workgroups (sequences x heads x tiles of rows x pieces), sequences x heads^2 under 2^32")
    qst, ost = _row_strides(T, HQ, Dh, qst, qt, "q"), (HQ * Dh, Dh) if o is None else _row_strides(T, HQ, Dh, o[1], qt, "out", True)
    return (T, HQ, B, qst, ost, (tstride, width), (B, T, max_q, HQ, HKV, Dh, scale, chunk, nchunk),
            T * HQ * nchunk if nchunk > 1 else 0, units * nchunk if rows > 64 else 0,
            (_rows(T, HQ, qst, 2, Dh), _rows(T, HQ, ost, 2, Dh), _rows(B, 1, (tstride, 0), 4, width), _rows(1, 1, (0, 0), 4, B),
             _rows(1, 1, (0, 0), 4, B + 1), _rows(NP, 1, (c0, 0), 1, HKV * page * Dh // 2),
             _rows(NP, 1, (s0, 0), 1, HKV * page * Dh // KV4_BLOCK)))


def kv4_attn(q, kc, ks, vc, vs, table, lens, sm_scale: float | None = None, cu_q=None, max_q: int = 1, out=None,
             max_len: int | None = None) -> torch.Tensor:
    """Causal attention of the newest tokens of every sequence over a 4-bit paged cache.
    q (T, HQ, D) bf16, HQ any multiple of the cache's heads; table (B, width) int32 page ids; lens (B,)
    int32 keys that the sequences hold, these tokens among them.  Tokens cu_q[b] .. cu_q[b + 1] - 1
    (cu_q (B + 1,) int32, 0 to T, not decreasing) are the last of sequence b, at most max_q of them; cu_q
    None: one token each.
    Token j of R sees keys 0 .. lens[b] - R + j; one that sees none gives 0.  max_len: a bound on lens
    that the caller knows (the table's width otherwise).  NaN: rows that need a page id outside of the
    cache, and those of sequences longer than their table row or than max_len (rounded up to whole pieces,
    kv4_chunk).  Rows of `out` that no sequence takes, and tokens past max_q, are left
    as they were (0 where the call makes it); `out` shares no memory with the other tensors.  Sums are held in
    fp32 and not divided before their end: values up to 2^80 are safe at any length.  Sequences are cut into
    pieces by kv4_chunk, more than 65535 of them not at all; at most 2^24 - 1 workgroups (a sequence's, by head,
    for 8, 16, 32 or, past 64 rows of a KV head, 128 rows each)."""
    i = _where(q, kc, ks, vc, vs, table, lens, cu_q, out)
    ps, where, HKV, Dh = _kv4_cache(kc, ks, vc, vs)
    T, HQ, B, qst, ost, tsz, sizes, parts, flags, lie = _attn_sizes(
        HKV, Dh, where, q.shape, q.stride(), q.dtype, table.shape, table.stride(), table.dtype, lens.shape, lens.stride(),
        lens.dtype, _m(cu_q), index(max_q), None if sm_scale is None else float(sm_scale),
        None if max_len is None else index(max_len), _m(out), kv4_chunk)
    _plain(q, out)
    qp = q.data_ptr()
    given = out is not None
    clear = out is None and cu_q is not None and parts > 0 and B > 0     # (by the join)
    if out is None:
        out = q.new_empty(T, HQ, Dh) if clear or cu_q is None else q.new_zeros(T, HQ, Dh)
    op = out.data_ptr()
    if T == 0 or B == 0:
        return out
    _aligned(qp | op)
    if given:
        lq, lo, lt, ll, lc, lw, ls = lie
        _apart("out", op, lo, (qp, lq), (table.data_ptr(), lt), (lens.data_ptr(), ll), (_ptr(cu_q) or 0, lc), (ps[0], lw), (ps[1], ls),
               (ps[2], lw), (ps[3], ls))
    wp = mp = fp = None
    if parts or flags:
        ws = q.new_empty(parts * (Dh + 2) + flags, dtype=torch.float32)
        wp = ws.data_ptr()
        mp = wp + 4 * parts * Dh
        fp = mp + 8 * parts
    _run(i, "oa_kv4_attn", qp, *qst, *ps, *where, table.data_ptr(), *tsz, lens.data_ptr(), _ptr(cu_q), *sizes, wp, mp, fp, op,
         *ost, clear)
    return out


# ================================================================== prefill index build
def qgs_codes(K, T: int, U, codes, scale, amax_ws, zc_ws=None) -> None:
    """a11 of one request: K (HKV, >=T, 128) bf16; U (HKV, 128, 32) fp32; codes (HKV, Lmax, 32)
    int8 (rows written up to T); scale (HKV, 32); amax_ws >= HKV*32 int32 scratch; zc_ws >= HKV*T*32
    fp32 scratch or None (then k U is formed twice; the same codes)."""
    dev = _dev(K, U, codes, scale, amax_ws)
    HKV = K.shape[0]
    _need(K.dtype == torch.bfloat16 and K.stride(-1) == 1, "K: bf16 with contiguous rows")
    _need(U.is_contiguous() and U.shape == (HKV, HEAD_DIM, RANK_Q), "U: (HKV, 128, 32) contiguous")
    _need(scale.is_contiguous() and scale.shape == (HKV, RANK_Q), "scale: (HKV, 32) contiguous")
    _need(codes.dtype == torch.int8 and codes.stride(2) == 1 and codes.stride(1) == RANK_Q,
          "codes: (HKV, Lmax, 32) int8 rows")
    _need(amax_ws.numel() >= HKV * RANK_Q, "amax_ws too small")
    _need(T <= K.shape[1] and T <= codes.shape[1], "T beyond the rows")
    if zc_ws is not None:
        _need(zc_ws.dtype == torch.float32 and zc_ws.is_contiguous() and zc_ws.numel() >= HKV * T * RANK_Q,
              "zc_ws: >= HKV*T*32 fp32, contiguous")
    lib.call("oa_qgs_codes", _ptr(K), K.stride(0), K.stride(1), HKV, T, _ptr(U), _ptr(codes),
             codes.stride(0), _ptr(scale), _ptr(amax_ws), _ptr(zc_ws), _stream(dev))


def query_metric(q, pick, cosv, sinv, scaling: float, mst_half, G: int, gm_out=None, m_out=None):
    """a10 metric of every query row of q (rows, Qn, 128) bf16 or fp32 (rows = KV rows * G):
    returns (gm_out (rows / G, 128, 128) group means, m_out (rows, 128, 128) metrics), fp32.
    pick (P,) int32 question positions; cosv, sinv (P, 128) fp64 RoPE cos / sin of each picked
    row's advance; mst_half (heads, 128, 128) fp32, used for row r as mst_half[r % heads]."""
    dev = _dev(q, pick, cosv, sinv, mst_half, gm_out, m_out)
    _need(q.dim() == 3 and q.shape[-1] == HEAD_DIM and q.stride(-1) == 1
          and q.dtype in (torch.bfloat16, torch.float32), "q: (rows, Qn, 128) bf16 or fp32, rows of dims contiguous")
    rows = q.shape[0]
    _need(rows % G == 0, "rows: a multiple of G")
    _need(pick.dtype == torch.int32 and pick.dim() == 1 and pick.is_contiguous(), "pick: (P,) int32")
    P = pick.numel()
    _need(1 <= P <= 64, "P: 1..64 picked rows")
    for t, nm in ((cosv, "cosv"), (sinv, "sinv")):
        _need(t.dtype == torch.float64 and t.shape == (P, HEAD_DIM) and t.is_contiguous(), f"{nm}: (P, 128) fp64")
    _need(mst_half.dtype == torch.float32 and mst_half.dim() == 3 and mst_half.shape[1:] == (HEAD_DIM, HEAD_DIM)
          and mst_half.is_contiguous(), "mst_half: (heads, 128, 128) fp32 contiguous")
    if gm_out is None:
        gm_out = torch.empty(rows // G, HEAD_DIM, HEAD_DIM, device=dev, dtype=torch.float32)
    if m_out is None:
        m_out = torch.empty(rows, HEAD_DIM, HEAD_DIM, device=dev, dtype=torch.float32)
    for t, n_, nm in ((gm_out, rows // G, "gm_out"), (m_out, rows, "m_out")):
        _need(t.dtype == torch.float32 and t.is_contiguous() and t.shape == (n_, HEAD_DIM, HEAD_DIM),
              f"{nm}: ({n_}, 128, 128) fp32 contiguous")
    lib.call("oa_query_metric", _ptr(q), int(q.dtype == torch.bfloat16), q.stride(0), q.stride(1), rows, G,
             _ptr(pick), P, _ptr(cosv), _ptr(sinv), float(scaling), _ptr(mst_half), mst_half.shape[0],
             _ptr(gm_out), _ptr(m_out), _stream(dev))
    return gm_out, m_out


def sym_eig_top(M, k: int, sweeps=None):
    """Top-k eigenpairs of symmetric positive semi-definite (batch, 128, 128) fp32 matrices (the
    lower triangle is read): (evals (batch, k), evecs (batch, 128, k)), ascending, the last k of
    torch.linalg.eigh's order; signs are free.  sweeps: (batch,) int32 or None, the Jacobi sweeps
    each matrix took (negative: unconverged at the cap)."""
    dev = _dev(M, sweeps)
    _need(M.dtype == torch.float32 and M.dim() == 3 and M.shape[1:] == (HEAD_DIM, HEAD_DIM)
          and M.stride(2) == 1 and M.stride(1) == HEAD_DIM
          and (M.shape[0] <= 1 or M.stride(0) >= HEAD_DIM * HEAD_DIM),
          "M: (batch, 128, 128) fp32 with contiguous matrices")
    _need(1 <= k <= 64, "k: 1..64")
    B = M.shape[0]
    m_stride = M.stride(0) if B > 1 else HEAD_DIM * HEAD_DIM
    if sweeps is not None:
        _need(sweeps.dtype == torch.int32 and sweeps.is_contiguous() and sweeps.numel() >= B,
              "sweeps: >= batch int32, contiguous")
    ev = torch.empty(B, k, device=dev, dtype=torch.float32)
    vec = torch.empty(B, HEAD_DIM, k, device=dev, dtype=torch.float32)
    if B:
        lib.call("oa_sym_eig_top", _ptr(M), m_stride, B, HEAD_DIM, k, _ptr(ev), _ptr(vec),
                 _ptr(sweeps), _stream(dev))
    return ev, vec


def qgc_project(K, T: int, W, G: int, zraw, colmean, zP=None, zmax=None) -> None:
    """a12 projection: zraw (HQ, T, 16) int16/bf16 = bf16(k W) (what kmeans_assign and
    kmeans_update read); colmean (HQ, 16); zP (HQ, T, 16) fp32 = bf16(k W) - colmean, or None; zmax
    (HQ, 16) int32 or None, the columns' bound words for kmeans_step."""
    dev = _dev(K, W, zraw, colmean, zmax)
    HQ = W.shape[0]
    _need(W.dtype == torch.bfloat16 and W.is_contiguous() and W.shape[1:] == (HEAD_DIM, RANK_C),
          "W: (HQ, 128, 16) bf16 contiguous")
    _need(K.shape[0] * G == HQ and T <= K.shape[1], "K: HQ / G rows of at least T tokens")
    _zraw(zraw, HQ, T)
    _need(colmean.is_contiguous() and colmean.shape == (HQ, RANK_C), "colmean: (HQ, 16) contiguous")
    if zP is not None:
        _need(zP.dtype == torch.float32 and zP.stride() == zraw.stride(), "zP: fp32, zraw's strides")
    ntiles = -(-T // 64)
    ws = torch.empty(HQ * ntiles * RANK_C, device=dev, dtype=torch.float64)
    args = (_ptr(K), K.stride(0), K.stride(1), HQ, G, T, _ptr(W), _ptr(zP), zraw.stride(0), _ptr(colmean), _ptr(ws),
            _ptr(zraw))
    if zmax is None:
        lib.call("oa_qgc_project", *args, _stream(dev))
        return
    _chk(zmax, "zmax", torch.int32, (HQ, RANK_C), contiguous=True)
    max_ws = torch.empty(HQ * -(-T // 512) * RANK_C, device=dev, dtype=torch.int32)
    lib.call("oa_qgc_project_max", *args, _ptr(max_ws), _ptr(zmax), _stream(dev))


def _zraw(zraw, HQ: int, T: int) -> None:
    _need(zraw.element_size() == 2 and zraw.dim() == 3 and zraw.shape[0] == HQ and zraw.shape[1] >= T
          and zraw.shape[2] == RANK_C and zraw.stride(2) == 1 and zraw.stride(1) == RANK_C,
          "zraw: (HQ, >=T, 16) 16-bit rows")


def kmeans_assign(zraw, colmean, T: int, cent, asg, asg8) -> None:
    """a12 assignment into asg (HQ, >=T) int32 and asg8 (HQ, >=T) uint8 rows; zP = zraw - colmean
    formed on the fly from the bf16 projection."""
    dev = _dev(zraw, colmean, cent, asg, asg8)
    HQ, C = cent.shape[0], cent.shape[1]
    _zraw(zraw, HQ, T)
    _need(colmean.is_contiguous() and colmean.shape == (HQ, RANK_C), "colmean: (HQ, 16) contiguous")
    _need(cent.is_contiguous() and cent.shape[2] == RANK_C, "cent: (HQ, C, 16) contiguous")
    _need(asg.stride(1) == 1 and asg8.stride(1) == 1, "asg rows must be contiguous")
    lib.call("oa_kmeans_assign", _ptr(zraw), _ptr(colmean), zraw.stride(0), HQ, T, _ptr(cent), C, _ptr(asg),
             asg.stride(0), _ptr(asg8), asg8.stride(0), _stream(dev))


def kmeans_step(zraw, colmean, T: int, init, cent, asg=None, asg8=None, ws=None, zmax=None) -> torch.Tensor:
    """kmeans_assign then kmeans_update's centroids (cent in place) without member lists; asg and asg8
    both None (not written) or both given.  ws: a byte workspace of a former call with the same sizes,
    or None; returns the workspace used.  zmax: qgc_project's bound words for this zraw and colmean, or
    None (zraw is then read once more for them)."""
    dev = _dev(zraw, colmean, cent, init, asg, asg8, ws, zmax)
    HQ, C = cent.shape[0], cent.shape[1]
    _zraw(zraw, HQ, T)
    _need(colmean.is_contiguous() and colmean.shape == (HQ, RANK_C), "colmean: (HQ, 16) contiguous")
    _need(cent.is_contiguous() and cent.shape[2] == RANK_C, "cent: (HQ, C, 16) contiguous")
    _need(init.dtype == torch.int32 and init.numel() == C and init.is_contiguous(), "init: (C,) int32")
    _need((asg is None) == (asg8 is None), "asg and asg8 are given together")
    if asg is not None:
        _chk(asg, "asg", torch.int32, (HQ, -T))
        _chk(asg8, "asg8", torch.uint8, (HQ, -T))
    need = lib.load().oa_kmeans_step_ws(HQ, T, C)
    _need(need > 0, "kmeans_step: rows, T and C must be positive, C at most 256")
    if ws is None or ws.numel() < need:
        ws = torch.empty(need, device=dev, dtype=torch.uint8)
    if zmax is not None:
        _chk(zmax, "zmax", torch.int32, (HQ, RANK_C), contiguous=True)
    lib.call("oa_kmeans_step_max", _ptr(zraw), _ptr(colmean), _ptr(zmax), zraw.stride(0), HQ, T, _ptr(cent), C,
             _ptr(init), _ptr(asg), 0 if asg is None else asg.stride(0), _ptr(asg8), 0 if asg8 is None else asg8.stride(0),
             _ptr(ws), ws.numel(), _stream(dev))
    return ws


def kmeans_update(zraw, colmean, T: int, asg8, init, cent, mem, cstart, clen, cnt=None) -> None:
    """a12 update of cent (HQ, C, 16) in place; init (C,) int32 initial positions; zP as in
    kmeans_assign; mem (HQ, >=T), cstart, clen (HQ, C) int32 receive the assignment's member lists."""
    dev = _dev(zraw, colmean, asg8, init, cent, mem, cstart, clen)
    HQ, C = cent.shape[0], cent.shape[1]
    _zraw(zraw, HQ, T)
    _need(colmean.is_contiguous() and colmean.shape == (HQ, RANK_C), "colmean: (HQ, 16) contiguous")
    _need(init.dtype == torch.int32 and init.numel() == C, "init: (C,) int32")
    _chk(mem, "mem", torch.int32, (HQ, -T))
    _chk(cstart, "cstart", torch.int32, (HQ, C), contiguous=True)
    _chk(clen, "clen", torch.int32, (HQ, C), contiguous=True)
    lib.call("oa_kmeans_update", _ptr(zraw), _ptr(colmean), zraw.stride(0), HQ, T, _ptr(asg8), asg8.stride(0),
             C, _ptr(init), _ptr(cent), _ptr(cnt), _ptr(mem), mem.stride(0), _ptr(cstart), _ptr(clen),
             _stream(dev))


def cluster_sums(K, V, T: int, G: int, C: int, nb, Sk, Sk2, Sv, mem, cstart, clen) -> None:
    """a13 over member lists already built (kmeans_update's for the assignment it was given):
    nb = clen, Sk/Sk2/Sv as cluster_build, which would sort that assignment again."""
    dev = _dev(K, V, nb, Sk, Sk2, Sv, mem, cstart, clen)
    HQ = nb.shape[0]
    _need(K.stride() == V.stride() and K.stride(-1) == 1, "K, V: same strides, contiguous rows")
    _need(K.shape[0] * G == HQ and T <= K.shape[1], "K: HQ / G rows of at least T tokens")
    for t, nm in ((nb, "nb"), (Sk, "Sk"), (Sk2, "Sk2"), (Sv, "Sv"), (cstart, "cstart"), (clen, "clen")):
        _need(t.is_contiguous(), f"{nm} must be contiguous")
    _need(mem.dtype == torch.int32 and mem.stride(-1) == 1 and cstart.dtype == torch.int32
          and clen.dtype == torch.int32, "mem, cstart, clen: int32")
    lib.call("oa_cluster_sums", _ptr(K), _ptr(V), K.stride(0), K.stride(1), HQ, G, T, C, _ptr(nb),
             _ptr(Sk), _ptr(Sk2), _ptr(Sv), _ptr(mem), mem.stride(0), _ptr(cstart), _ptr(clen),
             _stream(dev))


def cluster_build(K, V, T: int, G: int, asg8, C: int, nb, Sk, Sk2, Sv, mem, cstart, clen) -> None:
    """a13: nb (HQ, C), Sk/Sk2/Sv (HQ, C, 128), mem (HQ, >=T), cstart/clen (HQ, C)."""
    dev = _dev(K, V, asg8, nb, Sk, Sk2, Sv, mem, cstart, clen)
    HQ = nb.shape[0]
    _need(K.stride() == V.stride() and K.stride(-1) == 1, "K, V: same strides, contiguous rows")
    _need(K.shape[0] * G == HQ and T <= K.shape[1], "K: HQ / G rows of at least T tokens")
    for t, nm in ((nb, "nb"), (Sk, "Sk"), (Sk2, "Sk2"), (Sv, "Sv"), (cstart, "cstart"), (clen, "clen")):
        _need(t.is_contiguous(), f"{nm} must be contiguous")
    lib.call("oa_cluster_build", _ptr(K), _ptr(V), K.stride(0), K.stride(1), HQ, G, T, _ptr(asg8),
             asg8.stride(0), C, _ptr(nb), _ptr(Sk), _ptr(Sk2), _ptr(Sv), _ptr(mem), mem.stride(0),
             _ptr(cstart), _ptr(clen), _stream(dev))
