"""Thin torch-tensor wrappers over the per-kernel C ABI (used by the parity tests and the host-side model code).

Every function enqueues on torch's current HIP stream.  Tensors must live on the GPU; nothing here computes
on the host and nothing falls back to torch ops.
"""
import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import _lib as L
from ._lib import AttnDesc, GemmDesc, check, lib, ptr, stream_ptr

BF16 = torch.bfloat16


def _need(t, dtype=None):
    if not t.is_cuda:
        raise L.Vlt5Error("tensor must be on the GPU")
    if dtype is not None and t.dtype != dtype:
        raise L.Vlt5Error(f"expected {dtype}, got {t.dtype}")
    return t


def gemm(A, B, M, N, K, *, a_kmajor=False, b_kmajor=False, out=None, out_f32=False, alpha=1.0, bias=None, relu=False,
         resid=None, gate=None, gate_scale=1.0, drop_p=0.0, drop_seed=0, accum=False, split_k=1, tile=(0, 0),
         lda=None, ldb=None, ldc=None, batch=1, batch_strides=(0, 0, 0), emit=None, norm=None, tuning=None, relu_bits_out=None,
         gate_bits=None):
    """C[M,N] = epi(alpha * sum_k A[m,k] B[n,k]); A,B bf16 2-D tensors, k-major flags as in vlt5_gemm_desc.
    tuning: a vlt5_tuning record (_lib.make_tuning) for the launch's policy switches.
    emit = (w_norm f32 [N], xw bf16 [M,N], partials f32 [M,32]): producer side of a folded T5 RMS norm -- returns (out, nparts);
    norm = (partials, nparts, d, eps, rstd_out or None): consumer side."""
    g, out, _keep = gemm_desc(A, B, M, N, K, a_kmajor=a_kmajor, b_kmajor=b_kmajor, out=out, out_f32=out_f32, alpha=alpha, bias=bias,
                              relu=relu, resid=resid, gate=gate, gate_scale=gate_scale, drop_p=drop_p, drop_seed=drop_seed,
                              accum=accum, split_k=split_k, tile=tile, lda=lda, ldb=ldb, ldc=ldc, batch=batch,
                              batch_strides=batch_strides)
    if emit is not None:
        g.emit_norm_w, g.emit_xw_bf16, g.emit_partials = ptr(emit[0]), ptr(emit[1]), ptr(emit[2])
    if norm is not None:
        g.norm_partials, g.norm_nparts, g.norm_d, g.norm_eps, g.norm_rstd_out = ptr(norm[0]), norm[1], norm[2], norm[3], ptr(norm[4])
    if tuning is not None:
        g.tuning = C.pointer(tuning)
    if relu_bits_out is not None:          # uint8 [M, >= N/8]: the ReLU sign bits of the stored values (vlt5_gemm_desc.relu_bits_out)
        g.relu_bits_out, g.ld_bits = ptr(relu_bits_out), relu_bits_out.stride(0)
    if gate_bits is not None:              # ... and the same bits as the gate of a hidden-gradient GEMM, instead of `gate`
        g.gate_bits, g.ld_bits = ptr(gate_bits), gate_bits.stride(0)
    check(lib().vlt5_gemm_bf16(C.byref(g), stream_ptr()), "vlt5_gemm_bf16")
    if emit is not None:
        return out, g.emit_nparts
    return out


def gemm_desc(A, B, M, N, K, *, a_kmajor=False, b_kmajor=False, out=None, out_f32=False, alpha=1.0, bias=None, relu=False,
              resid=None, gate=None, gate_scale=1.0, drop_p=0.0, drop_seed=0, accum=False, split_k=1, tile=(0, 0),
              lda=None, ldb=None, ldc=None, batch=1, batch_strides=(0, 0, 0)):
    """The filled vlt5_gemm_desc of `gemm` without launching it: (desc, out, keep-alive) -- for launch loops that must not pay the
    descriptor construction per call (bench.py)."""
    _need(A, BF16), _need(B, BF16)
    if out is None:
        out = torch.empty(M, N, device=A.device, dtype=torch.float32 if out_f32 else BF16)
    out_f32 = out.dtype == torch.float32
    g = GemmDesc()
    g.A, g.B, g.C = ptr(A), ptr(B), ptr(out)
    g.M, g.N, g.K = M, N, K
    g.lda = lda if lda is not None else A.stride(0)
    g.ldb = ldb if ldb is not None else B.stride(0)
    g.ldc = ldc if ldc is not None else out.stride(0)
    g.a_kmajor, g.b_kmajor = int(a_kmajor), int(b_kmajor)
    g.alpha = alpha
    g.bias = ptr(bias)
    g.resid, g.ldr = ptr(resid), (resid.stride(0) if resid is not None else 0)
    g.gate, g.ldg, g.gate_scale = ptr(gate), (gate.stride(0) if gate is not None else 0), gate_scale
    g.drop_p, g.drop_seed = drop_p, drop_seed
    g.relu, g.out_f32, g.accum = int(relu), int(out_f32), int(accum)
    ws = None
    if split_k > 1:
        ws = torch.empty(lib().vlt5_gemm_workspace_bytes(M, g.ldc, split_k), device=A.device, dtype=torch.uint8)
        g.split_k, g.workspace = split_k, ptr(ws)
    g.tile_m, g.tile_n = tile
    g.batch = batch
    g.batch_stride_a, g.batch_stride_b, g.batch_stride_c = batch_strides
    return g, out, (A, B, ws, bias, resid, gate)


def layernorm_fwd(x, w, eps=1e-6, want_f32=False, drop_p=0.0, drop_seed=0):
    rows, d = x.shape
    yb = torch.empty(rows, d, device=x.device, dtype=BF16)
    yf = torch.empty(rows, d, device=x.device, dtype=torch.float32) if want_f32 else None
    rstd = torch.empty(rows, device=x.device, dtype=torch.float32)
    check(lib().vlt5_layernorm_fwd(ptr(_need(x, torch.float32)), ptr(w), ptr(yb), ptr(yf), ptr(rstd), rows, d, eps, drop_p,
                                   drop_seed, 0, 0, stream_ptr()), "vlt5_layernorm_fwd")
    return yb, yf, rstd


def layernorm_bwd(dy, x, w, rstd, dx=None, drop_p=0.0, drop_seed=0, want_bf16=False, dx_drop_p=0.0, dx_drop_seed=0,
                  deferred_reduce=False):
    rows, d = x.shape
    accum = dx is not None
    if dx is None:
        dx = torch.empty_like(x)
    dw = torch.empty(d, device=x.device, dtype=torch.float32)
    part = torch.empty(lib().vlt5_layernorm_bwd_blocks(rows), d, device=x.device, dtype=torch.float32)
    dxb = torch.empty(rows, d, device=x.device, dtype=BF16) if want_bf16 else None
    check(lib().vlt5_layernorm_bwd(ptr(dy), ptr(x), ptr(w), ptr(rstd), ptr(dx), ptr(None if deferred_reduce else dw), ptr(part),
                                   rows, d, int(accum), 0, drop_p, drop_seed, 0, 0, ptr(dxb), dx_drop_p, dx_drop_seed,
                                   stream_ptr()), "vlt5_layernorm_bwd")
    if deferred_reduce:                 # the engine's way: one multi-job reduction launch for many norms
        off = (L.c_ll * 1)(0)
        nb = (L.c_i * 1)(part.shape[0])
        check(lib().vlt5_colsum_multi(ptr(part), ptr(dw), off, nb, 1, part.shape[0], d, stream_ptr()), "vlt5_colsum_multi")
    if want_bf16:
        return dx, dw, dxb
    return dx, dw


def _attn_desc(q, k, v, H, dk, bias, key_mask, mask_value, causal, drop_p, drop_seed):
    B, Tq = q.shape[:2]
    Tk = k.shape[1]
    a = AttnDesc()
    a.q, a.k, a.v = ptr(_need(q, BF16)), ptr(_need(k, BF16)), ptr(_need(v, BF16))
    a.q_sb, a.q_st = q.stride(0), q.stride(1)
    a.k_sb, a.k_st = k.stride(0), k.stride(1)
    a.v_sb, a.v_st = v.stride(0), v.stride(1)
    if bias is not None:
        a.bias, a.bias_q, a.bias_k = ptr(bias), bias.shape[1], bias.shape[2]
    a.key_mask, a.mask_value, a.causal = ptr(key_mask), mask_value, int(causal)
    a.B, a.H, a.Tq, a.Tk, a.dk = B, H, Tq, Tk, dk
    a.drop_p, a.drop_seed = drop_p, drop_seed
    return a


def attn_fwd(q, k, v, H, dk, bias=None, key_mask=None, mask_value=-10000.0, causal=False, drop_p=0.0, drop_seed=0):
    """q [B,Tq,H*dk], k/v [B,Tk,H*dk] bf16 (any strides along batch/token) -> ctx [B,Tq,H*dk] bf16, lse [B,H,Tq]."""
    B, Tq = q.shape[:2]
    a = _attn_desc(q, k, v, H, dk, bias, key_mask, mask_value, causal, drop_p, drop_seed)
    ctx = torch.empty(B, Tq, H * dk, device=q.device, dtype=BF16)
    lse = torch.empty(B, H, Tq, device=q.device, dtype=torch.float32)
    a.ctx, a.o_sb, a.o_st, a.lse = ptr(ctx), ctx.stride(0), ctx.stride(1), ptr(lse)
    check(lib().vlt5_attn_fwd(C.byref(a), stream_ptr()), "vlt5_attn_fwd")
    return ctx, lse


def attn_bwd(q, k, v, d_ctx, lse, H, dk, bias=None, key_mask=None, mask_value=-10000.0, causal=False, drop_p=0.0,
             drop_seed=0, want_dbias=False):
    B, Tq = q.shape[:2]
    Tk = k.shape[1]
    a = _attn_desc(q, k, v, H, dk, bias, key_mask, mask_value, causal, drop_p, drop_seed)
    dq = torch.empty(B, Tq, H * dk, device=q.device, dtype=BF16)
    dk_ = torch.empty(B, Tk, H * dk, device=q.device, dtype=BF16)
    dv = torch.empty(B, Tk, H * dk, device=q.device, dtype=BF16)
    a.lse = ptr(lse)
    a.d_ctx, a.do_sb, a.do_st = ptr(_need(d_ctx, BF16)), d_ctx.stride(0), d_ctx.stride(1)
    a.dq, a.dq_sb, a.dq_st = ptr(dq), dq.stride(0), dq.stride(1)
    a.dk_, a.dk_sb, a.dk_st = ptr(dk_), dk_.stride(0), dk_.stride(1)
    a.dv, a.dv_sb, a.dv_st = ptr(dv), dv.stride(0), dv.stride(1)
    dbias = None
    if want_dbias and bias is not None:
        dbias = torch.zeros(B, H, bias.shape[1], bias.shape[2], device=q.device, dtype=torch.float32)
        a.dbias = ptr(dbias)
    check(lib().vlt5_attn_bwd(C.byref(a), stream_ptr()), "vlt5_attn_bwd")
    return dq, dk_, dv, dbias


def relbias_build(table, lut, H, Lq, Lk):
    bias = torch.empty(H, Lq, Lk, device=table.device, dtype=torch.float32)
    check(lib().vlt5_relbias_build(ptr(table), ptr(_need(lut, torch.int32)), ptr(bias), H, Lq, Lk, table.shape[0], stream_ptr()),
          "vlt5_relbias_build")
    return bias


def relbias_bwd(dS, lut, nbuckets):
    nmat, H, Lq, Lk = dS.shape
    dtable = torch.empty(nbuckets, H, device=dS.device, dtype=torch.float32)
    scratch = torch.empty(64 * H * Lq * Lk, device=dS.device, dtype=torch.float32)
    check(lib().vlt5_relbias_bwd(ptr(dS), ptr(lut), ptr(dtable), ptr(scratch), nmat, H, Lq, Lk, nbuckets, 0, stream_ptr()),
          "vlt5_relbias_bwd")
    return dtable


def cast_bf16(src, dst=None):
    if dst is None:
        dst = torch.empty(src.shape, device=src.device, dtype=BF16)
    check(lib().vlt5_cast_bf16(ptr(_need(src, torch.float32)), ptr(dst), src.numel(), stream_ptr()), "vlt5_cast_bf16")
    return dst


def ce_fwd(logits, labels):
    R, V = logits.shape
    loss = torch.empty(R, device=logits.device, dtype=torch.float32)
    lse = torch.empty(R, device=logits.device, dtype=torch.float32)
    check(lib().vlt5_ce_fwd(ptr(_need(logits, torch.float32)), ptr(_need(labels, torch.int64)), ptr(loss), ptr(lse), R, V,
                            stream_ptr()), "vlt5_ce_fwd")
    return loss, lse


def loss_reduce(loss_tok, labels, scores):
    B, T = labels.shape
    loss = torch.empty(1, device=labels.device, dtype=torch.float32)
    row_w = torch.empty(B * T, device=labels.device, dtype=torch.float32)
    check(lib().vlt5_loss_reduce(ptr(loss_tok), ptr(labels), ptr(scores), ptr(loss), ptr(row_w), B, T, stream_ptr()),
          "vlt5_loss_reduce")
    return loss, row_w


def ce_bwd(logits, labels, lse, row_w, gout=None):
    R, V = logits.shape
    d = torch.empty(R, V, device=logits.device, dtype=BF16)
    check(lib().vlt5_ce_bwd(ptr(logits), ptr(labels), ptr(lse), ptr(row_w), ptr(gout), ptr(d), R, V, stream_ptr()), "vlt5_ce_bwd")
    return d


def proto_pool(hidden, S, split):
    """hidden f32 [B, >=S, d] (batch stride may exceed S*d) -> poolQ, poolV [B,d]."""
    B, d = hidden.shape[0], hidden.shape[2]
    pq = torch.empty(B, d, device=hidden.device, dtype=torch.float32)
    pv = torch.empty(B, d, device=hidden.device, dtype=torch.float32)
    check(lib().vlt5_proto_pool(ptr(_need(hidden, torch.float32)), hidden.stride(0), B, S, d, split, ptr(pq), ptr(pv), stream_ptr()),
          "vlt5_proto_pool")
    return pq, pv


def proto_class_mean(pool, onehot):
    B, d = pool.shape
    Cn = onehot.shape[1]
    proto = torch.empty(Cn, d, device=pool.device, dtype=torch.float32)
    cnt = torch.empty(Cn, device=pool.device, dtype=torch.float32)
    onehot = _need(onehot.contiguous(), torch.float32)       # held in a local until the launch is enqueued
    check(lib().vlt5_proto_class_mean(ptr(pool), ptr(onehot), ptr(proto), ptr(cnt), B, Cn, d, stream_ptr()),
          "vlt5_proto_class_mean")
    return proto, cnt


def proto_retrieve(protos, pool, out_f32=None, sb=0, out_bf16=None, sb_bf16=0):
    B, d = pool.shape
    idx = torch.empty(B, device=pool.device, dtype=torch.int64)
    scratch = torch.empty(protos.shape[0], d, device=pool.device, dtype=torch.float32)
    check(lib().vlt5_proto_retrieve(ptr(_need(protos, torch.float32)), ptr(pool), ptr(idx), ptr(out_f32), sb, ptr(out_bf16), sb_bf16,
                                    ptr(scratch), B, protos.shape[0], d, stream_ptr()), "vlt5_proto_retrieve")
    return idx


def proto_memory_loss(pool, onehot, protos):
    out = torch.empty(1, device=pool.device, dtype=torch.float32)
    onehot = onehot.contiguous()
    check(lib().vlt5_proto_memory_loss(ptr(pool), ptr(onehot), ptr(protos), ptr(out), pool.shape[0], protos.shape[0],
                                       pool.shape[1], stream_ptr()), "vlt5_proto_memory_loss")
    return out


def drop_cast(src, drop_p=0.0, drop_seed=0):
    """bf16(dropout(src)) with the engine's counter-based mask (element index = row*cols + col)."""
    rows, cols = src.shape
    dst = torch.empty(rows, cols, device=src.device, dtype=BF16)
    check(lib().vlt5_drop_cast(ptr(_need(src, torch.float32)), ptr(dst), rows, cols, drop_p, drop_seed, stream_ptr()), "vlt5_drop_cast")
    return dst


def glu_fwd(u, ff, drop_p=0.0, drop_seed=0):
    """u bf16 [rows, 2*ff] -> h bf16 [rows, ff] = dropout(gelu_new(u[:, :ff]) * u[:, ff:])  (HF T5DenseGatedActDense)."""
    rows = u.shape[0]
    h = torch.empty(rows, ff, device=u.device, dtype=BF16)
    check(lib().vlt5_glu_fwd(ptr(_need(u, BF16)), ptr(h), rows, ff, drop_p, drop_seed, stream_ptr()), "vlt5_glu_fwd")
    return h


def glu_bwd(dh, u, ff, drop_p=0.0, drop_seed=0):
    rows = u.shape[0]
    du = torch.empty(rows, 2 * ff, device=u.device, dtype=BF16)
    check(lib().vlt5_glu_bwd(ptr(_need(dh, BF16)), ptr(_need(u, BF16)), ptr(du), rows, ff, drop_p, drop_seed, stream_ptr()), "vlt5_glu_bwd")
    return du


def qkv_attn_fwd(xn, wqkv, B, S, H, bias=None, key_mask=None, mask_value=-10000.0, drop_p=0.0, drop_seed=0):
    """Fused q|k|v projection + attention core (csrc/enc_attn.hip): xn bf16 [B*S, d], wqkv bf16 [3*H*64, d] ->
    qkv bf16 [B, S, 3*H*64], ctx bf16 [B, S, H*64], lse f32 [B, H, S]."""
    d = xn.shape[1]
    inner = H * 64
    qkv = torch.empty(B, S, 3 * inner, device=xn.device, dtype=BF16)
    a = _attn_desc(qkv[:, :, :inner], qkv[:, :, inner:2 * inner], qkv[:, :, 2 * inner:], H, 64, bias, key_mask, mask_value, False,
                   drop_p, drop_seed)
    ctx = torch.empty(B, S, inner, device=xn.device, dtype=BF16)
    lse = torch.empty(B, H, S, device=xn.device, dtype=torch.float32)
    a.ctx, a.o_sb, a.o_st, a.lse = ptr(ctx), ctx.stride(0), ctx.stride(1), ptr(lse)
    check(lib().vlt5_qkv_attn_fwd(ptr(_need(xn, BF16)), ptr(_need(wqkv, BF16)), ptr(qkv), C.byref(a), d, stream_ptr()), "vlt5_qkv_attn_fwd")
    return qkv, ctx, lse


def dec_attn_fused(xn, w, wo, B, T, H, k=None, v=None, bias=None, key_mask=None, mask_value=-10000.0, drop_p=0.0, drop_seed=0):
    """Fused decoder attention sublayer between the norms (csrc/dec_attn.hip).  Self-attention (k is None): w = [3*H*64, d] q|k|v rows,
    causal; cross-attention: w = [H*64, d] q rows, k / v = projected encoder-side keys / values [B, Tk, H*64] (any batch / token strides).
    xn bf16 [B*T, d], wo bf16 [d, H*64] -> (proj bf16 [B, T, 3*H*64] or [B, T, H*64], ctx bf16 [B, T, H*64], lse f32 [B, H, T],
    slabs f32 [H, B*T, d]: slab h = that head's share of the output projection)."""
    from ._lib import DecAttnDesc
    d = xn.shape[1]
    inner = H * 64
    dev = xn.device
    cross = k is not None
    proj = torch.empty(B, T, inner if cross else 3 * inner, device=dev, dtype=BF16)
    if cross:
        a = _attn_desc(proj, k, v, H, 64, bias, key_mask, mask_value, False, drop_p, drop_seed)
    else:
        a = _attn_desc(proj[:, :, :inner], proj[:, :, inner:2 * inner], proj[:, :, 2 * inner:], H, 64, bias, key_mask, mask_value, True,
                       drop_p, drop_seed)
    ctx = torch.empty(B, T, inner, device=dev, dtype=BF16)
    lse = torch.empty(B, H, T, device=dev, dtype=torch.float32)
    slabs = torch.empty(H, B * T, d, device=dev, dtype=torch.float32)
    a.ctx, a.o_sb, a.o_st, a.lse = ptr(ctx), ctx.stride(0), ctx.stride(1), ptr(lse)
    e = DecAttnDesc()
    e.xn_bf16, e.w_bf16, e.wo_bf16, e.proj_bf16 = ptr(_need(xn, BF16)), ptr(_need(w, BF16)), ptr(_need(wo, BF16)), ptr(proj)
    e.o_slabs, e.slab_stride, e.d_model, e.core = ptr(slabs), B * T * d, d, a
    fn = lib().vlt5_cross_attn_fwd if cross else lib().vlt5_dec_self_attn_fwd
    check(fn(C.byref(e), stream_ptr()), "vlt5_cross_attn_fwd" if cross else "vlt5_dec_self_attn_fwd")
    return proj, ctx, lse, slabs


def enc_attn_sublayer(x, ln_w, wqkv, wo, B, S, H, bias=None, key_mask=None, mask_value=-10000.0, eps=1e-6, drop_p=0.0, seeds=(0, 0)):
    """Forward of the whole encoder self-attention sublayer through `vlt5_enc_attn_fwd` (norm, fused q|k|v projection + core, output
    projection with dropout + residual).  x f32 [B*S, d]; wqkv bf16 [3*H*64, d]; wo bf16 [d, H*64].  Returns (x_out, saved) where
    `saved` feeds `enc_attn_sublayer_bwd`."""
    from ._lib import EncAttnDesc
    d = x.shape[1]
    inner = H * 64
    dev = x.device
    sv = dict(x=x, ln_w=ln_w, wqkv=wqkv, wo=wo, bias=bias, key_mask=key_mask,
              xn=torch.empty(B * S, d, device=dev, dtype=BF16), rstd=torch.empty(B * S, device=dev, dtype=torch.float32),
              qkv=torch.empty(B * S, 3 * inner, device=dev, dtype=BF16), ctx=torch.empty(B * S, inner, device=dev, dtype=BF16),
              lse=torch.empty(B, H, S, device=dev, dtype=torch.float32))
    out = torch.empty_like(x)
    e = EncAttnDesc()
    e.x, e.ln_w, e.wqkv_bf16, e.wo_bf16, e.x_out = ptr(_need(x, torch.float32)), ptr(ln_w), ptr(_need(wqkv, BF16)), ptr(_need(wo, BF16)), ptr(out)
    e.xn_bf16, e.rstd, e.qkv_bf16, e.ctx_bf16, e.lse = ptr(sv["xn"]), ptr(sv["rstd"]), ptr(sv["qkv"]), ptr(sv["ctx"]), ptr(sv["lse"])
    if bias is not None:
        e.bias, e.bias_q, e.bias_k = ptr(bias), bias.shape[1], bias.shape[2]
    e.key_mask, e.mask_value = ptr(key_mask), mask_value
    e.B, e.S, e.H, e.d_model, e.eps = B, S, H, d, eps
    e.drop_p, e.seed_probs, e.seed_out = drop_p, seeds[0], seeds[1]
    check(lib().vlt5_enc_attn_fwd(C.byref(e), stream_ptr()), "vlt5_enc_attn_fwd")
    sv["desc"] = e
    return out, sv


def enc_attn_sublayer_bwd(dy, sv, want_dscores=False):
    """Backward through `vlt5_enc_attn_bwd`: returns dx, d_wqkv, d_wo, d_ln_w (f32) and, optionally, the per-sample bias-block gradient."""
    from ._lib import EncAttnGrads
    e = sv["desc"]
    dev = dy.device
    g = EncAttnGrads()
    dx = torch.empty_like(dy)
    dwqkv = torch.empty(sv["wqkv"].shape, device=dev, dtype=torch.float32)
    dwo = torch.empty(sv["wo"].shape, device=dev, dtype=torch.float32)
    dln = torch.empty(sv["ln_w"].shape, device=dev, dtype=torch.float32)
    ds = None
    if want_dscores and sv["bias"] is not None:
        ds = torch.zeros(e.B, e.H, e.bias_q, e.bias_k, device=dev, dtype=torch.float32)
    ws = torch.empty(lib().vlt5_enc_attn_bwd_workspace_bytes(e.B, e.S, e.H, e.d_model), device=dev, dtype=torch.uint8)
    g.dy, g.dx, g.d_wqkv, g.d_wo, g.d_ln_w, g.d_scores = ptr(_need(dy, torch.float32)), ptr(dx), ptr(dwqkv), ptr(dwo), ptr(dln), ptr(ds)
    check(lib().vlt5_enc_attn_bwd(C.byref(e), C.byref(g), ptr(ws), stream_ptr()), "vlt5_enc_attn_bwd")
    return dx, dwqkv, dwo, dln, ds


# ---- the token-step in low precision: 4-bit weights, a paged key/value cache, the attention over it -------------------------------
FP8, F32, I32 = torch.float8_e4m3fn, torch.float32, torch.int32
_KV_TYPE = {BF16: 0, torch.int8: 1, FP8: 2}
_F32_ZERO = 2.0 ** -150                # the largest number that f32 rounds to 0 (half its smallest, a tie)


class W4Weight(NamedTuple):
    """A weight [N, K] in four bits: codes uint8 [N, K/2] (two e2m1 codes a byte, the even k in the low bits), scales bf16
    [N, ceil(K/group)], one for `group` (32, 64 or 128) consecutive k.  Made by `quant_w4`."""
    codes: torch.Tensor
    scales: torch.Tensor
    group: int


class KVPages(NamedTuple):
    """The paged key/value cache of one layer: k, v [pages, kv heads, page size, d_kv] (bf16, int8 or float8_e4m3fn) and, for the 8-bit
    types, k_scale, v_scale f32 [pages, kv heads, page size].  Made by `kv_pages`."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: Optional[torch.Tensor] = None
    v_scale: Optional[torch.Tensor] = None


def _here(t):
    """(device index, raw current stream) of the current device, on which `t` has to be (the library launches on the current device)."""
    i = t.get_device()
    if i < 0:
        raise L.Vlt5Error("tensor must be on the GPU")
    if i != torch._C._cuda_getDevice():
        raise L.Vlt5Error(f"tensor on {t.device}, but cuda:{torch._C._cuda_getDevice()} is the current device")
    return i, torch._C._cuda_getCurrentRawStream(i)


def _refuse(dev, *want):
    """Raises for the first (name, tensor, dtypes, shape, contiguous) that is not so: what a call's one combined check found to be wrong."""
    for name, t, dtypes, shape, contiguous in want:
        if t is None:
            raise L.Vlt5Error(f"{name} is missing")
        got = f"got {t.dtype} {tuple(t.shape)} with strides {tuple(t.stride())} on {t.device}"
        if t.device != dev or t.dtype not in dtypes or t.dim() != len(shape) or any(s is not None and s != n for s, n in zip(shape, t.shape)):
            raise L.Vlt5Error(f"{name}: expected {' or '.join(map(str, dtypes))} {shape} on {dev}, {got}")
        if not t.is_contiguous() if contiguous else t.stride(-1) != 1 and t.shape[-1] > 1:
            raise L.Vlt5Error(f"{name}: expected {'a contiguous tensor' if contiguous else 'unit column stride'}, {got}")
    raise L.Vlt5Error("sizes do not fit together: " + ", ".join(f"{n} {tuple(t.shape)}" for n, t, *_ in want))


def _row_stride(t, rows, cols):
    """Row stride of a 2-D tensor; that of a single row, which torch leaves arbitrary, is made up."""
    return t.stride(0) if rows > 1 else (cols + 7) // 8 * 8


def quant_w4(w, group=128):
    """A weight [N, K] (f32 or bf16, unit column stride, K a multiple of 32) as a `W4Weight`."""
    dev = w.device
    _, st = _here(w)
    if w.dim() != 2 or w.dtype not in (BF16, torch.float32) or w.stride(1) != 1:
        _refuse(dev, ("w", w, (BF16, torch.float32), (None, None), False))
    N, K = w.shape
    if group not in (32, 64, 128):
        raise L.Vlt5Error(f"group: 32, 64 or 128, got {group}")
    codes = torch.empty(N, K // 2, device=dev, dtype=torch.uint8)
    scales = torch.empty(N, -(-K // group), device=dev, dtype=BF16)
    f32 = w.dtype == torch.float32
    check(lib().vlt5_quant_w4(w.data_ptr() if f32 else None, None if f32 else w.data_ptr(), _row_stride(w, N, K), N, K, group, codes.data_ptr(),
                              scales.data_ptr(), st), "vlt5_quant_w4")
    return W4Weight(codes, scales, group)


def decode_linear_w4(x, w, *, alpha=1.0, resid=None, relu=False, out_f32=False, out=None):
    """act(alpha * x W^T (+ resid)) for a few rows x bf16 [rows <= 256, K] against a `W4Weight`; resid f32 [rows, N]; alpha not 0 in f32.  Returns
    bf16, or f32 with out_f32; `out` takes the result instead (its type decides; it may be `resid` itself, and may
    share no memory with anything else)."""
    codes, scales, group = w
    dev = x.device
    at, st = _here(x)
    if group not in (32, 64, 128):
        raise L.Vlt5Error(f"group: 32, 64 or 128, got {group}")
    if -_F32_ZERO <= alpha <= _F32_ZERO:                                             # (0 in the descriptor, which the library takes for 1)
        raise L.Vlt5Error(f"alpha: {alpha} is 0 in f32, and 0 is not a factor")
    if x.dim() != 2 or codes.dim() != 2:
        _refuse(dev, ("x", x, (BF16,), (None, None), False), ("codes", codes, (torch.uint8,), (None, None), True))
    (rows, K), (N, K2) = x.shape, codes.shape
    groups = -(-K // group)
    if (x.dtype is not BF16 or x.stride(1) != 1 or K != 2 * K2 or codes.dtype is not torch.uint8 or codes.get_device() != at or not codes.is_contiguous()
            or scales.dtype is not BF16 or scales.get_device() != at or scales.shape != (N, groups) or not scales.is_contiguous()):
        _refuse(dev, ("x", x, (BF16,), (None, 2 * K2), False), ("codes", codes, (torch.uint8,), (N, K2), True), ("scales", scales, (BF16,), (N, groups), True))
    if out is None:
        out = torch.empty(rows, N, device=dev, dtype=torch.float32 if out_f32 else BF16)
        f32, ldo = out_f32, N
    else:
        f32 = out.dtype is torch.float32
        if not (f32 or out.dtype is BF16) or out.shape != (rows, N) or out.device != dev or (N > 1 and out.stride(1) != 1):
            _refuse(dev, ("out", out, (BF16, torch.float32), (rows, N), False))
        ldo = out.stride(0) if rows > 1 else N
    rp, ldr = None, 0
    if resid is not None:
        if resid.dtype is not torch.float32 or resid.shape != (rows, N) or resid.device != dev or (N > 1 and resid.stride(1) != 1):
            _refuse(dev, ("resid", resid, (torch.float32,), (rows, N), False))
        rp, ldr = resid.data_ptr(), resid.stride(0) if rows > 1 else N
    if rows:
        o = out.data_ptr()
        d = L.DecodeLinearW4Desc(x.data_ptr(), _row_stride(x, rows, K), codes.data_ptr(), scales.data_ptr(), rows, N, K, group, alpha, None if f32 else o, ldo,
                                 o if f32 else None, ldo, rp, ldr, relu, None, 0)
        if 2 * min(rows, 16) * K >= L.W4_SPLIT_BYTES:                                # (below, the reduction stays within a workgroup)
            need = lib().vlt5_decode_linear_w4_workspace_bytes(rows, N, K)
            if need > 0:
                ws = torch.empty(need, device=dev, dtype=torch.uint8)
                d.workspace, d.workspace_bytes = ws.data_ptr(), need
        check(lib().vlt5_decode_linear_w4(C.byref(d), st), "vlt5_decode_linear_w4")
    return out


def kv_pages(n_pages, n_kv_heads, d_kv, page_size=64, dtype=torch.int8, device="cuda"):
    """An empty paged cache: bf16, int8 or float8_e4m3fn."""
    if dtype not in _KV_TYPE:
        raise L.Vlt5Error(f"kv_pages: bf16, int8 or float8_e4m3fn, got {dtype}")
    shape = (n_pages, n_kv_heads, page_size, d_kv)
    k, v = (torch.zeros(shape, device=device, dtype=torch.uint8 if dtype == FP8 else dtype).view(dtype) for _ in range(2))
    if dtype == BF16:
        return KVPages(k, v)
    return KVPages(k, v, *(torch.zeros(shape[:3], device=device, dtype=torch.float32) for _ in range(2)))


def _paged(cache, table, kv_lens, cu_q, n_tok, max_q, at, dev):
    """The cache and the sequences of a call as the library takes them."""
    k, v, ks, vs = cache
    dtype = k.dtype
    kind = _KV_TYPE.get(dtype)
    if kind is None or k.dim() != 4 or table.dim() != 2:
        _refuse(dev, ("cache.k", k, tuple(_KV_TYPE), (None,) * 4, True), ("block table", table, (torch.int32,), (None, None), True))
    shape = k.shape
    B, mp = table.shape
    if v.dtype is not dtype or v.shape != shape or k.get_device() != at or v.get_device() != at or not k.is_contiguous() or not v.is_contiguous():
        _refuse(dev, ("cache.k", k, (dtype,), tuple(shape), True), ("cache.v", v, (dtype,), tuple(shape), True))
    n, h, page, d = shape
    ksp = vsp = None
    if kind:
        rows = (n, h, page)
        if (ks is None or vs is None or ks.dtype is not F32 or vs.dtype is not F32 or ks.shape != rows or vs.shape != rows or ks.get_device() != at
                or vs.get_device() != at or not ks.is_contiguous() or not vs.is_contiguous()):
            _refuse(dev, ("cache.k_scale", ks, (torch.float32,), rows, True), ("cache.v_scale", vs, (torch.float32,), rows, True))
        ksp, vsp = ks.data_ptr(), vs.data_ptr()
    if (table.dtype is not I32 or table.get_device() != at or not table.is_contiguous() or kv_lens.dtype is not I32 or kv_lens.get_device() != at
            or kv_lens.shape != (B,) or not kv_lens.is_contiguous()):
        _refuse(dev, ("block table", table, (torch.int32,), (B, mp), True), ("kv_lens", kv_lens, (torch.int32,), (B,), True))
    cu = None
    if cu_q is None:
        max_q = 1
        if n_tok != B and n_tok:
            raise L.Vlt5Error(f"{n_tok} tokens for {B} sequences: without cu_q every sequence has one")
    else:
        if cu_q.dtype is not I32 or cu_q.get_device() != at or cu_q.shape != (B + 1,) or not cu_q.is_contiguous():
            _refuse(dev, ("cu_q", cu_q, (torch.int32,), (B + 1,), True))
        cu = cu_q.data_ptr()
    return (L.PagedKV(k.data_ptr(), v.data_ptr(), ksp, vsp, n, h, d, page, kind), L.PagedSeqs(table.data_ptr(), kv_lens.data_ptr(), cu, B, mp, n_tok, max_q or 0),
            h, d, B)


def kv_page_write(cache, k, v, table, kv_lens, *, cu_q=None, max_q=None):
    """New keys | values k, v bf16 [tokens, kv heads * d_kv] (any token stride) into the pages of their sequences, quantised on the way.

    table i32 [B, pages of a sequence], kv_lens i32 [B]: keys of every sequence with the new tokens counted; cu_q i32 [B + 1]: first new
    token of every sequence (None: one token each); max_q: the most new tokens any of them has (None: as if one had them all, which costs
    workgroups that find nothing to do).  A page id outside the cache = not there."""
    dev = k.device
    at, st = _here(k)
    if k.dim() != 2:
        _refuse(dev, ("k", k, (BF16,), (None, None), False))
    n, width = k.shape
    kv, seqs, h, d, _ = _paged(cache, table, kv_lens, cu_q, n, max_q, at, dev)
    if k.dtype is not BF16 or v.dtype is not BF16 or width != h * d or v.shape != (n, width) or v.get_device() != at or k.stride(1) != 1 or v.stride(1) != 1:
        _refuse(dev, ("k", k, (BF16,), (None, h * d), False), ("v", v, (BF16,), (n, h * d), False))
    if n:
        check(lib().vlt5_kv_page_write(C.byref(kv), C.byref(seqs), k.data_ptr(), _row_stride(k, n, width), v.data_ptr(), _row_stride(v, n, width), st), "vlt5_kv_page_write")


def kv_page_read(cache, table, kv_lens, T):
    """Positions 0 .. T-1 of every sequence back as (k, v) bf16 [B, T, kv heads * d_kv], zeros at and past its length: what `attn_fwd` takes."""
    dev = cache.k.device
    at, st = _here(cache.k)
    kv, seqs, h, d, B = _paged(cache, table, kv_lens, None, 0, None, at, dev)
    k = torch.empty(B, T, h * d, device=dev, dtype=BF16)
    v = torch.empty(B, T, h * d, device=dev, dtype=BF16)
    if T and B:
        check(lib().vlt5_kv_page_read(C.byref(kv), C.byref(seqs), T, k.data_ptr(), v.data_ptr(), st), "vlt5_kv_page_read")
    return k, v


def paged_attn(q, cache, table, kv_lens, *, cu_q=None, max_q=None, max_kv=None, scale=1.0, causal=True, rel_bias=None, out=None, want_lse=False):
    """softmax(scale * q K^T + bias) V of the newest tokens, q bf16 [tokens, heads * d_kv] (any token stride), over the pages of their
    sequences, whose keys are written already (table, kv_lens, cu_q, max_q as in `kv_page_write`).

    heads: any multiple of the cache's; scale > 0; causal: a token sees the positions up to its own, else all keys; rel_bias f32 [heads, n]: added by
    how far the key lies back, its last column for everything further (T5's decoder bias); max_kv: about the longest length, for the split
    of the work only.  A token that sees no key gets zeros; rows of `out` that belong to no sequence keep what they hold.  `out` may be
    `q` itself and otherwise shares no memory with it.
    Returns out bf16 [tokens, heads * d_kv], with want_lse also f32 [tokens, heads] (-inf without keys)."""
    dev = q.device
    at, st = _here(q)
    if q.dim() != 2:
        _refuse(dev, ("q", q, (BF16,), (None, None), False))
    n, width = q.shape
    kv, seqs, h, d, _ = _paged(cache, table, kv_lens, cu_q, n, max_q, at, dev)
    if q.dtype is not BF16 or width % (h * d) or not width or q.stride(1) != 1:
        raise L.Vlt5Error(f"q: expected bf16 rows of a multiple of {h} heads of {d}, got {q.dtype} {tuple(q.shape)} with strides {tuple(q.stride())}")
    H = width // d
    if out is None:
        out, o_st = torch.empty(n, width, device=dev, dtype=BF16), width
    else:
        if out.dtype is not BF16 or out.shape != (n, width) or out.device != dev or out.stride(1) != 1:
            _refuse(dev, ("out", out, (BF16,), (n, width), False))
        o_st = _row_stride(out, n, width)
    lse = torch.empty(n, H, device=dev, dtype=torch.float32) if want_lse else None
    bias, nd = None, 0
    if rel_bias is not None:
        if not causal or rel_bias.dim() != 2 or rel_bias.shape[0] != H or rel_bias.shape[1] < 1 or rel_bias.dtype is not torch.float32 or rel_bias.device != dev \
                or not rel_bias.is_contiguous():
            raise L.Vlt5Error(f"rel_bias: contiguous f32 [{H}, distances] of a causal call, got {rel_bias.dtype} {tuple(rel_bias.shape)} on {rel_bias.device}, causal={causal}")
        bias, nd = rel_bias.data_ptr(), rel_bias.shape[1]
    if n:
        l = lib()
        desc = L.PagedAttnDesc(kv, seqs, q.data_ptr(), _row_stride(q, n, width), out.data_ptr(), o_st, None if lse is None else lse.data_ptr(), bias, nd, H, scale,
                               causal, max_kv or 0, None, 0)
        ref = C.byref(desc)
        if seqs.max_pages * kv.page_size >= L.PAGED_SHARED_KV and not 0 < desc.max_kv < L.PAGED_SHARED_KV:      # (below, the keys of a row are not shared out)
            need = l.vlt5_paged_attn_workspace_bytes(ref)
            if need > 0:
                ws = torch.empty(need, device=dev, dtype=torch.uint8)
                desc.workspace, desc.workspace_bytes = ws.data_ptr(), need
        check(l.vlt5_paged_attn(ref, st), "vlt5_paged_attn")
    return (out, lse) if want_lse else out
