"""The operator surface on CUDA tensors, one function per C-ABI entry point.

Names and argument meanings follow the reference's operators
(`llm/ref_model.py` DeviceModel: quant_act, linear, rmsnorm; `llm/compile_model.py`
ModelCompiler: embed, attention, ffn_up; `llm/runtime.py` Sampler). Every call
runs on the current torch CUDA stream and raises W8A8Error on a nonzero status.
Tensors are passed as raw device pointers; torch only owns the memory.
"""
import ctypes
import functools
from typing import NamedTuple

import numpy as np
import torch

from . import _lib

F32, I8, I32 = torch.float32, torch.int8, torch.int32
SFU_EXP, SFU_RECIP, SFU_RSQRT, SFU_SILU, SFU_GELU = 0, 1, 2, 3, 4
ACTS = {"silu": 0, "gelu_tanh": 1}


def _p(t):
    return None if t is None else t.data_ptr()


def _st():
    return torch.cuda.current_stream().cuda_stream


def _need(t, dtype, name):
    if not t.is_cuda or t.dtype != dtype or not t.is_contiguous():
        raise ValueError(f"{name}: a contiguous CUDA {dtype} tensor is required, got {t.dtype} on {t.device}")


def sfu(func, x, out=None):
    _need(x, F32, "x")
    out = torch.empty_like(x) if out is None else out
    _lib.check("w8a8_sfu", _lib.load().w8a8_sfu(func, _p(x), _p(out), x.numel(), _st()))
    return out


def quant_act(x):
    """x [rows, k] fp32 -> (xq int8 [rows, k], s_x [rows])."""
    _need(x, F32, "x")
    x2 = x.reshape(-1, x.shape[-1])
    xq = torch.empty(x2.shape, dtype=I8, device=x.device)
    s = torch.empty(x2.shape[0], dtype=F32, device=x.device)
    _lib.check("w8a8_quant_act", _lib.load().w8a8_quant_act(_p(x2), x2.shape[0], x2.shape[1], _p(xq), _p(s), _st()))
    return xq.reshape(x.shape), s


def rmsnorm(x, g, eps):
    _need(x, F32, "x")
    x2 = x.reshape(-1, x.shape[-1])
    y = torch.empty_like(x2)
    _lib.check("w8a8_rmsnorm", _lib.load().w8a8_rmsnorm(_p(x2), _p(g), x2.shape[0], x2.shape[1], float(eps), _p(y),
                                                       _st()))
    return y.reshape(x.shape)


def embed(tokens, emb_q, emb_s, out=None):
    m, (vocab, dim) = tokens.numel(), emb_q.shape
    out = torch.empty(m, dim, dtype=F32, device=emb_q.device) if out is None else out
    _lib.check("w8a8_embed", _lib.load().w8a8_embed(_p(tokens), m, _p(emb_q), _p(emb_s), vocab, dim, _p(out),
                                                   _st()))
    return out


def error_flags():
    """Read and clear the device error flags (bit 0: an out-of-range token;
    w8a8.h lists the others)."""
    v = ctypes.c_uint32(0)
    _lib.check("w8a8_error_flags", _lib.load().w8a8_error_flags(ctypes.byref(v)))
    return v.value


def linear(xq, s_x, w, s_w, out=None, acc=None, resid=None):
    """W8A8 linear on int8 rows: y = (f32(xq . W^T) * s_w) * s_x [+ resid]."""
    _need(xq, I8, "xq")
    _need(w, I8, "w")
    m, k = xq.shape
    n = w.shape[0]
    out = torch.empty(m, n, dtype=F32, device=w.device) if out is None else out
    _lib.check("w8a8_linear", _lib.load().w8a8_linear(_p(xq), _p(s_x), m, k, _p(w), _p(s_w), n, _p(resid), _p(out),
                                                     _p(acc), _st()))
    return out


def linear_fused(x, w, s_w, norm_g=None, eps=0.0, resid=None, out=None, s_x_out=None):
    """[rmsnorm ->] quant_act -> linear [-> + resid] on fp32 rows x [m, k]."""
    _need(x, F32, "x")
    _need(w, I8, "w")
    m, k = x.shape
    n = w.shape[0]
    out = torch.empty(m, n, dtype=F32, device=w.device) if out is None else out
    _lib.check("w8a8_linear_fused", _lib.load().w8a8_linear_fused(
        _p(x), _p(norm_g), float(eps), m, k, _p(w), _p(s_w), n, _p(resid), _p(out), _p(s_x_out), _st()))
    return out


def linear_chain(x, w, s_w, norm_g=None, eps=0.0, x_amax=None, resid=None, out=None, clear=None):
    """The decode chain's fused linear: quant_act(x) with max|x| posted by the
    producer (x_amax), or rmsnorm + quant_act; `clear` zeroed after the wait."""
    _need(x, F32, "x")
    m, k = x.shape
    n = w.shape[0]
    out = torch.empty(m, n, dtype=F32, device=x.device) if out is None else out
    _lib.check("w8a8_linear_chain", _lib.load().w8a8_linear_chain(
        _p(x), _p(norm_g), float(eps), _p(x_amax), m, k, _p(w), _p(s_w), n, _p(resid), _p(out), _p(clear),
        0 if clear is None else clear.numel(), _st()))
    return out


def ffn_swiglu_chain(x, norm_g, eps, w_gate, s_gate, w_up, s_up, h, h_amax, clear=None):
    """The decode chain's SwiGLU: h and max|h| per row posted into h_amax."""
    m, k = x.shape
    _lib.check("w8a8_ffn_swiglu_chain", _lib.load().w8a8_ffn_swiglu_chain(
        _p(x), _p(norm_g), float(eps), m, k, _p(w_gate), _p(s_gate), _p(w_up), _p(s_up), w_gate.shape[0], _p(h),
        _p(h_amax), _p(clear), 0 if clear is None else clear.numel(), _st()))
    return h


def ffn_scratch(rows, device):
    n = _lib.load().w8a8_ffn_scratch_bytes(rows)
    return torch.zeros(n, dtype=torch.uint8, device=device)


def ffn_swiglu(x, norm_g, eps, w_gate, s_gate, w_up, s_up, scratch, h=None, h_q=None, s_h=None, requant=True,
               act="silu"):
    """Decode SwiGLU dispatch: returns (h fp32, h_q int8, s_h); with
    requant=False only h (h_q, s_h None; the down projection quantizes h).
    act: the gate, "silu" or "gelu_tanh"."""
    _need(x, F32, "x")
    m, k = x.shape
    hidden = w_gate.shape[0]
    dev = x.device
    h = torch.empty(m, hidden, dtype=F32, device=dev) if h is None else h
    if requant:
        h_q = torch.empty(m, hidden, dtype=I8, device=dev) if h_q is None else h_q
        s_h = torch.empty(m, dtype=F32, device=dev) if s_h is None else s_h
    else:
        h_q = s_h = scratch = None
    _lib.check("w8a8_ffn_gated", _lib.load().w8a8_ffn_gated(
        _p(x), _p(norm_g), float(eps), m, k, _p(w_gate), _p(s_gate), _p(w_up), _p(s_up), hidden, ACTS[act], _p(h),
        _p(h_q), _p(s_h), _p(scratch), 0 if scratch is None else scratch.numel(), _st()))
    return h, h_q, s_h


def quant_rows(x, norm_g=None, eps=0.0, xq=None, s_x=None):
    """int8 rows and scales of x (quant_act, after rmsnorm when norm_g is given)."""
    _need(x, F32, "x")
    m, k = x.shape
    xq = torch.empty(m, k, dtype=I8, device=x.device) if xq is None else xq
    s_x = torch.empty(m, dtype=F32, device=x.device) if s_x is None else s_x
    _lib.check("w8a8_quant_rows", _lib.load().w8a8_quant_rows(_p(x), _p(norm_g), float(eps), m, k, _p(xq), _p(s_x),
                                                              _st()))
    return xq, s_x


def gemm(xq, s_x, w, s_w, out=None, acc=None, resid=None):
    """Tensor-core W8A8 linear for any row count (same results as linear())."""
    m, k = xq.shape
    n = w.shape[0]
    out = torch.empty(m, n, dtype=F32, device=xq.device) if out is None else out
    _lib.check("w8a8_gemm", _lib.load().w8a8_gemm(_p(xq), _p(s_x), m, k, _p(w), _p(s_w), n, _p(resid), _p(out),
                                                  _p(acc), _st()))
    return out


def gemm_swiglu(xq, s_x, w_gate, s_gate, w_up, s_up, out=None, act="silu"):
    """Tensor-core gated pair: h = act(g) * u for any row count (act "silu"
    or "gelu_tanh")."""
    m, k = xq.shape
    n = w_gate.shape[0]
    out = torch.empty(m, n, dtype=F32, device=xq.device) if out is None else out
    _lib.check("w8a8_gemm_gated", _lib.load().w8a8_gemm_gated(_p(xq), _p(s_x), m, k, _p(w_gate), _p(s_gate),
                                                              _p(w_up), _p(s_up), n, ACTS[act], _p(out), _st()))
    return out


def moe_scratch(rows, dim, top_k, expert_hidden, device):
    n = _lib.load().w8a8_moe_scratch_bytes(rows, dim, top_k, expert_hidden)
    return torch.zeros(n, dtype=torch.uint8, device=device)


def moe_ffn(x, norm_g, eps, router_q, router_s, top_k, gate_q, gate_s, up_q, up_s, down_q, down_s, scratch,
            resid=None, out=None, ids=None, w=None):
    """MoE FFN rows (hf_generic.QMixtralMoe): returns (y = resid + moe(rmsnorm(x)),
    ids [rows, top_k] int32, w [rows, top_k] fp32). resid defaults to x; out may
    be resid (in place)."""
    _need(x, F32, "x")
    m, dim = x.shape
    experts, ih = router_q.shape[0], gate_q.shape[1]
    dev = x.device
    resid = x if resid is None else resid
    out = torch.empty(m, dim, dtype=F32, device=dev) if out is None else out
    ids = torch.empty(m, top_k, dtype=torch.int32, device=dev) if ids is None else ids
    w = torch.empty(m, top_k, dtype=F32, device=dev) if w is None else w
    _lib.check("w8a8_moe_ffn", _lib.load().w8a8_moe_ffn(
        _p(x), _p(norm_g), float(eps), m, dim, _p(router_q), _p(router_s), experts, top_k, _p(gate_q), _p(gate_s),
        _p(up_q), _p(up_s), ih, _p(down_q), _p(down_s), _p(resid), _p(out), _p(ids), _p(w), _p(scratch),
        scratch.numel(), _st()))
    return out, ids, w


def moe_ffn_ep(x, norm_g, eps, router_q, router_s, top_k, expert_lo, gate_q, gate_s, up_q, up_s, down_q, down_s,
               scratch, wy, ids, w):
    """Expert parallelism: the MoE FFN rows over this rank's experts
    [expert_lo, expert_lo + gate_q.shape[0]); wy [rows, top_k, dim] receives
    w_j * y_j of their slots and +0 for the others."""
    _need(x, F32, "x")
    m, dim = x.shape
    experts, (local, ih) = router_q.shape[0], gate_q.shape[:2]
    _lib.check("w8a8_moe_ffn_ep", _lib.load().w8a8_moe_ffn_ep(
        _p(x), _p(norm_g), float(eps), m, dim, _p(router_q), _p(router_s), experts, top_k, int(expert_lo), local,
        _p(gate_q), _p(gate_s), _p(up_q), _p(up_s), ih, _p(down_q), _p(down_s), _p(wy), _p(ids), _p(w),
        _p(scratch), scratch.numel(), _st()))
    return wy


MOE_MAX_ROWS = 4096


def moe_rows_scratch(rows, dim, experts, top_k, expert_hidden, device):
    n = _lib.load().w8a8_moe_rows_scratch_bytes(rows, dim, experts, top_k, expert_hidden)
    return torch.zeros(n, dtype=torch.uint8, device=device)


def moe_ffn_rows(x, norm_g, eps, router_q, router_s, top_k, gate_q, gate_s, up_q, up_s, down_q, down_s, scratch,
                 resid=None, out=None, ids=None, w=None, expert_lo=0, wy=None):
    """moe_ffn (wy None) or moe_ffn_ep (wy given, expert_lo: this rank's first
    expert) for many rows at once, the pairs grouped by expert; scratch from
    moe_rows_scratch."""
    _need(x, F32, "x")
    m, dim = x.shape
    experts, (local, ih) = router_q.shape[0], gate_q.shape[:2]
    dev = x.device
    if wy is None:
        resid = x if resid is None else resid
        out = torch.empty(m, dim, dtype=F32, device=dev) if out is None else out
    ids = torch.empty(m, top_k, dtype=torch.int32, device=dev) if ids is None else ids
    w = torch.empty(m, top_k, dtype=F32, device=dev) if w is None else w
    _lib.check("w8a8_moe_ffn_rows", _lib.load().w8a8_moe_ffn_rows(
        _p(x), _p(norm_g), float(eps), m, dim, _p(router_q), _p(router_s), experts, top_k, int(expert_lo), local,
        _p(gate_q), _p(gate_s), _p(up_q), _p(up_s), ih, _p(down_q), _p(down_s), _p(resid), _p(out), _p(wy),
        _p(ids), _p(w), _p(scratch), scratch.numel(), _st()))
    return (out if wy is None else wy), ids, w


def moe_combine(wy, resid, out):
    """out = resid + the k-order fold of wy [rows, top_k, dim]."""
    m, k, dim = wy.shape
    _lib.check("w8a8_moe_combine", _lib.load().w8a8_moe_combine(_p(wy), m, k, dim, _p(resid), _p(out), _st()))
    return out


def attn_scratch(rows, heads, kv_heads, head_dim, seq_len, device):
    n = _lib.load().w8a8_attn_scratch_bytes(rows, heads, kv_heads, head_dim, seq_len)
    return torch.zeros(n, dtype=torch.uint8, device=device)


VARIANTS = {"norm": 0, "qsum": 1}


def attn_args(cfg, rows, pos, qkv, kc, vc, att, consts, cos, sin, scratch, q_norm=None, k_norm=None, att_amax=None,
              ch=None):
    """The W8A8AttnArgs block of one layer (kept alive by the caller: a CUDA
    graph replays the pointers it captured). ch: the per-channel KV constants
    (device tensors k_scale / inv_sk_ch, inv_sv_ch / a_v_ch) or None."""
    inv_sk, inv_sv, a_k, a_v = consts
    ch = ch or {}
    return _lib.W8A8AttnArgs(
        rows=rows, heads=cfg.heads, kv_heads=cfg.kv_heads, head_dim=cfg.head_dim, seq_len=cfg.seq_len,
        variant=VARIANTS[cfg.attn], pos=_p(pos), qkv=_p(qkv), q_norm=_p(q_norm), k_norm=_p(k_norm),
        eps=float(np.float32(cfg.eps)), rope_cos=_p(cos), rope_sin=_p(sin), inv_sk=float(inv_sk),
        inv_sv=float(inv_sv), a_k=float(a_k), a_v=float(a_v), k_cache=_p(kc), v_cache=_p(vc), att=_p(att),
        scratch=_p(scratch), scratch_bytes=scratch.numel(), att_amax=_p(att_amax), k_scale=_p(ch.get("k_scale")),
        inv_sk_ch=_p(ch.get("inv_sk_ch")), inv_sv_ch=_p(ch.get("inv_sv_ch")), a_v_ch=_p(ch.get("a_v_ch")))


def attn(args):
    import ctypes
    _lib.check("w8a8_attn", _lib.load().w8a8_attn(ctypes.byref(args), _st()))


def kv_append(args):
    """Every row's K / V (args.rows rows, any number) into the cache."""
    _lib.check("w8a8_kv_append", _lib.load().w8a8_kv_append(ctypes.byref(args), _st()))


def attn_prefill(args):
    """The attention of all args.rows rows (their K / V appended before) in one launch."""
    _lib.check("w8a8_attn_prefill", _lib.load().w8a8_attn_prefill(ctypes.byref(args), _st()))


def attn_batch(args, slots, slot_stride):
    """Batched decode attention: slot b = row b of pos / qkv / att, caches at
    + b * slot_stride bytes (args built for one row and slot 0's caches)."""
    import ctypes
    _lib.check("w8a8_attn_batch", _lib.load().w8a8_attn_batch(ctypes.byref(args), slots, slot_stride, _st()))


def argmax(logits, out=None):
    m, n = logits.reshape(-1, logits.shape[-1]).shape
    out = torch.empty(m, dtype=I32, device=logits.device) if out is None else out
    _lib.check("w8a8_argmax", _lib.load().w8a8_argmax(_p(logits), m, n, _p(out), _st()))
    return out


def classifier(x, w, s_w, norm_g, eps, out=None, argmax_key=None):
    """Final rmsnorm -> quant_act -> classifier GEMV [+ fused greedy argmax key]."""
    _need(x, F32, "x")
    m, k = x.shape
    n = w.shape[0]
    out = torch.empty(m, n, dtype=F32, device=w.device) if out is None else out
    _lib.check("w8a8_classifier", _lib.load().w8a8_classifier(
        _p(x), _p(norm_g), float(eps), m, k, _p(w), _p(s_w), n, _p(out), _p(argmax_key), _st()))
    return out


def key_token(key):
    """The token index packed in an argmax key (host side)."""
    return 0xFFFFFFFF - (int(key) & 0xFFFFFFFF)


def decode_advance(tokens, pos, argmax_key, rows, next_token=None):
    _lib.check("w8a8_decode_advance", _lib.load().w8a8_decode_advance(
        _p(tokens), _p(pos), _p(argmax_key), _p(next_token), rows, _st()))


# ------------------------------------------------------------- tensor parallel
def tp_embed(comm, tokens, emb_q, emb_s, out):
    """w8a8_embed that also starts a tensor-parallel step (advances the epoch)."""
    m, (vocab, dim) = tokens.numel(), emb_q.shape
    _lib.check("w8a8_tp_embed", _lib.load().w8a8_tp_embed(ctypes.byref(comm), _p(tokens), m, _p(emb_q), _p(emb_s),
                                                         vocab, dim, _p(out), _st()))
    return out


def tp_linear(args):
    """One decode GEMV of a rank's shard (a prepared W8A8TpLinearArgs)."""
    _lib.check("w8a8_tp_linear", _lib.load().w8a8_tp_linear(ctypes.byref(args), _st()))


def tp_attn(args, comm, amax_out):
    _lib.check("w8a8_tp_attn", _lib.load().w8a8_tp_attn(ctypes.byref(args), ctypes.byref(comm), amax_out, _st()))


def tp_advance(comm, keys, tokens, pos, rows, next_token=None):
    _lib.check("w8a8_tp_advance", _lib.load().w8a8_tp_advance(ctypes.byref(comm), keys, _p(tokens), _p(pos),
                                                             _p(next_token), rows, _st()))


def tp_seed(comm, keys, token):
    _lib.check("w8a8_tp_seed", _lib.load().w8a8_tp_seed(ctypes.byref(comm), keys, int(token), _st()))


def tp_moe_ffn(comm, x, norm_g, eps, router_q, router_s, top_k, expert_lo, gate_q, gate_s, up_q, up_s, down_q,
               down_s, scratch, terms, ids, w):
    """Expert parallelism over the exchange: the terms of this rank's experts'
    slots into every rank's `terms` block (decode rows)."""
    _need(x, F32, "x")
    m, dim = x.shape
    experts, (local, ih) = router_q.shape[0], gate_q.shape[:2]
    _lib.check("w8a8_tp_moe_ffn", _lib.load().w8a8_tp_moe_ffn(
        ctypes.byref(comm), _p(x), _p(norm_g), float(eps), m, dim, _p(router_q), _p(router_s), experts, top_k,
        int(expert_lo), local, _p(gate_q), _p(gate_s), _p(up_q), _p(up_s), ih, _p(down_q), _p(down_s), terms,
        _p(ids), _p(w), _p(scratch), scratch.numel(), _st()))


def tp_moe_combine(comm, terms, rows, top_k, resid, out):
    dim = resid.shape[-1]
    _lib.check("w8a8_tp_moe_combine", _lib.load().w8a8_tp_moe_combine(ctypes.byref(comm), terms, rows, top_k, dim,
                                                                     _p(resid), _p(out), _st()))
    return out


def row_amax(x, out):
    """max|x| per row as float bits (int32 tensor [rows])."""
    m, k = x.shape
    _lib.check("w8a8_row_amax", _lib.load().w8a8_row_amax(_p(x), m, k, _p(out), _st()))
    return out


def quant_rows_posted(x, amax, xq, s_x):
    """quant_act of x rows with the given max|x| bits."""
    m, k = x.shape
    _lib.check("w8a8_quant_rows_posted", _lib.load().w8a8_quant_rows_posted(_p(x), _p(amax), m, k, _p(xq), _p(s_x),
                                                                           _st()))
    return xq, s_x


def dequant_resid(acc, s_x, s_w, out, resid=None):
    """out = [resid +] (f32(acc) * s_w) * s_x over int32 rows acc [rows, n]."""
    m, n = acc.shape
    _lib.check("w8a8_dequant_resid", _lib.load().w8a8_dequant_resid(_p(acc), _p(s_x), _p(s_w), m, n, _p(resid),
                                                                   _p(out), _st()))
    return out



# ------------------------------------------------- block-scaled 8-bit KV cache
class KvBlocks(NamedTuple):
    """One layer's cache in 8 bits with a scale per (slot, KV head, block of
    tokens): codes k, v int8 [slots, kv_heads, capacity, head_dim] and scales
    k_scale, v_scale fp32 [slots, kv_heads, capacity / block]; a value is
    code * scale of its block. The kvb_ calls take any such 4-tuple; the slot
    dimension may be strided (one layer of a [slots, layers, ...] cache)."""
    k: torch.Tensor
    k_scale: torch.Tensor
    v: torch.Tensor
    v_scale: torch.Tensor


_KVB_TYPES = {F32: 0, torch.bfloat16: 1, torch.float16: 2}
KVB_BLOCKS = (16, 32, 64, 128)


def kvb_cache(slots, kv_heads, capacity, head_dim, block=64, device="cuda"):
    """An empty cache; capacity is rounded up to whole blocks."""
    if block not in KVB_BLOCKS:
        raise ValueError(f"block {block}: one of {KVB_BLOCKS}")
    blocks = -(-capacity // block)
    codes = lambda: torch.zeros(slots, kv_heads, blocks * block, head_dim, dtype=I8, device=device)
    scales = lambda: torch.zeros(slots, kv_heads, blocks, dtype=F32, device=device)
    return KvBlocks(codes(), scales(), codes(), scales())


@functools.lru_cache(maxsize=256)
def _kvb_layout(k, ks, v, vs, strides, name):
    """What a cache's shapes and strides (None: all contiguous) say: slots,
    heads, capacity, head_dim, block, slot strides (a refused one raises)."""
    if len(k) != 4 or v != k or len(ks) != 3 or ks[:2] != k[:2] or vs != ks or ks[2] == 0 or k[2] % ks[2]:
        raise ValueError(f"{name}: codes {tuple(k)} / {tuple(v)} and scales {tuple(ks)} / {tuple(vs)} do not belong "
                         "together")
    S, H, T, D = k
    NB = ks[2]
    if strides is None:
        return S, H, T, D, T // NB, H * T * D, H * NB
    k_st, ks_st, v_st, vs_st = strides
    if k_st[1:] != (T * D, D, 1) or v_st[1:] != k_st[1:] or ks_st[1:] != (NB, 1) or vs_st[1:] != ks_st[1:] or \
            (S > 1 and (v_st != k_st or vs_st != ks_st)):
        raise ValueError(f"{name}: each slot's codes and scales must be contiguous, K's and V's alike")
    return S, H, T, D, T // NB, k_st[0], ks_st[0]


def _kvb(cache, name="cache"):
    """The checked W8A8KvBlocks of a cache, and its device's index."""
    k, ks, v, vs = cache
    if k.dtype != I8 or v.dtype != I8 or ks.dtype != F32 or vs.dtype != F32:
        raise ValueError(f"{name}: int8 codes and fp32 scales are required")
    dense = k.is_contiguous() and ks.is_contiguous() and v.is_contiguous() and vs.is_contiguous()
    layout = _kvb_layout(k.shape, ks.shape, v.shape, vs.shape,
                         None if dense else (k.stride(), ks.stride(), v.stride(), vs.stride()), name)
    dev = k.get_device()
    if not k.is_cuda or ks.get_device() != dev or v.get_device() != dev or vs.get_device() != dev:
        raise ValueError(f"{name}: CUDA tensors on one device are required")
    return _lib.W8A8KvBlocks(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), *layout), dev


def _kvb_index(t, n, dev, name):
    if t.dtype != I32 or t.shape != (n,) or t.get_device() != dev or not t.is_contiguous():
        raise ValueError(f"{name}: a contiguous int32 [{n}] tensor on cuda:{dev} is required")


def _kvb_rows(t, heads, hd, dev, name):
    """(dtype code, elements between rows) of rows [rows, heads, hd] whose rows
    are contiguous (a slice of a wider row is fine)."""
    code, sh, st = _KVB_TYPES.get(t.dtype), t.shape, t.stride()
    if code is None or len(sh) != 3 or t.get_device() != dev:
        raise ValueError(f"{name}: fp32, bf16 or fp16 [rows, {heads or 'heads'}, {hd}] on cuda:{dev} is required")
    if sh[2] != hd or (heads and sh[1] != heads) or st[2] != 1 or (sh[1] > 1 and st[1] != hd):
        raise ValueError(f"{name}: [rows, {heads or 'heads'}, {hd}] with contiguous rows is required, got {tuple(sh)} "
                         f"with strides {st}")
    return code, st[0] if sh[0] > 1 else sh[1] * hd


def _kvb_mass(t, k, name="mass"):
    if t.dtype != F32 or t.shape != k.shape[:3] or not t.is_contiguous() or t.get_device() != k.get_device():
        raise ValueError(f"{name}: a contiguous fp32 {tuple(k.shape[:3])} tensor on {k.device} is required")


def _kvb_call(fn, dev, *args):
    """One C call on the current stream of device dev (made current for it)."""
    if dev == torch._C._cuda_getDevice():
        rc = getattr(_lib.load(), fn)(*args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            rc = getattr(_lib.load(), fn)(*args, torch._C._cuda_getCurrentRawStream(dev))
    if rc:
        _lib.check(fn, rc)


def kvb_append(k, v, cache, pos, start=None):
    """Rows k, v [rows, kv_heads, head_dim] into the cache: slot b's rows
    start[b] .. start[b + 1] - 1 (start None: row b) at positions pos[b] on
    (negative: an idle slot). A block's scale grows with its largest value; its
    older codes are rescaled with it. The slot ends with its last row: tokens it
    held behind it are lost."""
    c, dev = _kvb(cache)
    dt, ks = _kvb_rows(k, c.kv_heads, c.head_dim, dev, "k")
    dv, vs = _kvb_rows(v, c.kv_heads, c.head_dim, dev, "v")
    if dt != dv or k.shape[0] != v.shape[0]:
        raise ValueError("k and v: the same type and number of rows are required")
    _kvb_index(pos, c.slots, dev, "pos")
    if start is not None:
        _kvb_index(start, c.slots + 1, dev, "start")
    _kvb_call("w8a8_kvb_append", dev, ctypes.byref(c), k.data_ptr(), ks, v.data_ptr(), vs, dt, k.shape[0],
              pos.data_ptr(), None if start is None else start.data_ptr())


def kvb_read(cache, pos, start, rows, dtype=F32, k=None, v=None):
    """The values held at the rows' positions: k, v [rows, kv_heads, head_dim]
    (zeros for idle slots; rows behind the last sequence are left alone)."""
    c, dev = _kvb(cache)
    _kvb_index(pos, c.slots, dev, "pos")
    if start is not None:
        _kvb_index(start, c.slots + 1, dev, "start")
    if dtype not in _KVB_TYPES or rows < 0:
        raise ValueError(f"dtype {dtype}, rows {rows}: fp32, bf16 or fp16 and a row count are required")
    H, D = c.kv_heads, c.head_dim
    for t, name in ((k, "k"), (v, "v")):
        if t is not None and (t.shape != (rows, H, D) or not t.is_contiguous() or t.get_device() != dev or
                              t.dtype != dtype):
            raise ValueError(f"{name}: a contiguous {dtype} {(rows, H, D)} tensor is required")
    k = torch.empty_strided((rows, H, D), (H * D, D, 1), dtype=dtype, device=dev) if k is None else k
    v = torch.empty_like(k) if v is None else v
    _kvb_call("w8a8_kvb_read", dev, ctypes.byref(c), rows, pos.data_ptr(),
              None if start is None else start.data_ptr(), k.data_ptr(), v.data_ptr(), _KVB_TYPES[dtype])
    return k, v


@functools.lru_cache(maxsize=256)
def _kvb_scratch_bytes(layout, heads, rows, one_row, mass, dtype):
    # sizes alone decide; the pointers are never followed
    c = _lib.W8A8KvBlocks(256, 256, 256, 256, *layout)
    return _lib.load().w8a8_kvb_attn_scratch_bytes(ctypes.byref(c), heads, rows, one_row, mass, dtype)


def kvb_attn_scratch(cache, heads, rows, start=True, mass=False, dtype=F32):
    """Scratch for kvb_attn (start False) or kvb_attn_rows (True) calls of at
    most `rows` rows; one per call that may overlap another."""
    c, dev = _kvb(cache)
    n = _lib.load().w8a8_kvb_attn_scratch_bytes(ctypes.byref(c), heads, rows, int(not start), int(mass),
                                                _KVB_TYPES[dtype])
    return torch.empty(n, dtype=torch.uint8, device=dev)


def _kvb_attn(q, cache, pos, start, scale, mass, out, scratch):
    c, dev = _kvb(cache)
    dt, qs = _kvb_rows(q, 0, c.head_dim, dev, "q")
    rows, heads, hd = q.shape
    _kvb_index(pos, c.slots, dev, "pos")
    if start is not None:
        _kvb_index(start, c.slots + 1, dev, "start")
    if mass is not None:
        _kvb_mass(mass, cache[0])
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous() or out.get_device() != dev:
        raise ValueError(f"out: a contiguous {q.dtype} {tuple(q.shape)} tensor is required")
    if scratch is None:
        n = _kvb_scratch_bytes((c.slots, c.kv_heads, c.capacity, c.head_dim, c.block, c.slot_stride, c.scale_stride),
                               heads, rows, int(start is None), int(mass is not None), dt)
        scratch = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    elif scratch.get_device() != dev or scratch.dtype != torch.uint8 or not scratch.is_contiguous():
        raise ValueError(f"scratch: contiguous bytes on cuda:{dev} are required")
    _kvb_call("w8a8_kvb_attn", dev, ctypes.byref(c), q.data_ptr(), qs, dt, heads, rows, pos.data_ptr(),
              None if start is None else start.data_ptr(), hd ** -0.5 if scale is None else scale, out.data_ptr(),
              None if mass is None else mass.data_ptr(), None if scratch is None else scratch.data_ptr(),
              0 if scratch is None else scratch.numel())
    return out


def kvb_attn(q, cache, pos, scale=None, mass=None, out=None, scratch=None):
    """Decode attention over the cache: row b of q [slots, heads, head_dim]
    attends slot b's tokens 0 .. pos[b] (its own appended before); a negative
    pos gives a zero row, a NaN or an infinity in a head's query NaN. scale:
    1 / sqrt(head_dim) by default. mass (fp32 [slots, kv_heads, capacity]): each token's probabilities, summed over the
    query heads of its KV head, are added to it. scratch: kvb_attn_scratch()
    bytes of this call's own, or None to take them from torch's allocator."""
    return _kvb_attn(q, cache, pos, None, scale, mass, out, scratch)


def kvb_attn_rows(q, cache, pos, start, scale=None, mass=None, out=None, scratch=None):
    """Prompt attention over the cache: slot b's rows start[b] .. start[b + 1]
    - 1 of q [rows, heads, head_dim] stand at positions pos[b], pos[b] + 1, ...
    and attend the tokens up to their own (all appended before). Rows behind
    the last sequence are left as they are in `out`; the rest as kvb_attn. Scores of
    up to 2^24 in size (past 2^27 a row may become NaN)."""
    if start is None:
        raise ValueError("start: an int32 [slots + 1] tensor is required")
    return _kvb_attn(q, cache, pos, start, scale, mass, out, scratch)


def kvb_evict(cache, mass, count, keep, sink=0, recent=0, dst=None, dst_mass=None):
    """Cut every slot that holds more than `keep` tokens (count [slots]) to
    `keep`: the first `sink`, the last `recent` and the heaviest by `mass` of
    those between, moved together in their order; in place, or into dst /
    dst_mass. From then on a token's place is not its position: append and attend
    at places (the new length is the next one). Returns (kept [slots, kv_heads, keep] int32: each place's former
    position, -1 past the new length; the new lengths [slots] int32)."""
    c, dev = _kvb(cache)
    _kvb_mass(mass, cache[0])
    _kvb_index(count, c.slots, dev, "count")
    d = None
    if dst is not None:
        d, ddev = _kvb(dst, "dst")
        if dst_mass is None:
            raise ValueError("dst_mass: required with dst")
        _kvb_mass(dst_mass, dst[0], "dst_mass")
        if ddev != dev:
            raise ValueError(f"dst: a cache on cuda:{dev} is required")
    elif dst_mass is not None:
        raise ValueError("dst_mass: only with dst")
    if not 0 < keep <= c.capacity:
        raise ValueError(f"keep {keep}: 1 .. {c.capacity}")
    H = c.kv_heads
    kept = torch.empty_strided((c.slots, H, keep), (H * keep, keep, 1), dtype=I32, device=dev)
    left = torch.empty_like(count)
    _kvb_call("w8a8_kvb_evict", dev, ctypes.byref(c), mass.data_ptr(), count.data_ptr(), keep, sink, recent,
              None if d is None else ctypes.byref(d), None if d is None else dst_mass.data_ptr(), kept.data_ptr(),
              left.data_ptr())
    return kept, left
