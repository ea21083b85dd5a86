"""`torch.ops.w8a8.*`: the main operators of the C ABI registered with
torch.library, for callers that hold torch tensors (the host side of the
reference's `llm/compile_model.py` dispatches: quant_act, the W8A8 linear,
RMSNorm, the fused SwiGLU, embedding, the classifier; `llm/sa_funcsim.py`'s
SFU). Each op allocates its outputs and calls the same C entry point as
`ops.py` on the current stream; a fake (meta) implementation gives the output
shapes for tracing. Importing this module registers them:

    import torch2riscv_accelerator_b200.torch_ops
    xq, s_x = torch.ops.w8a8.quant_act(x)
    y = torch.ops.w8a8.linear(xq, s_x, w, s_w)

There is no CPU kernel: on a CPU tensor the C ABI refuses the call.
"""
import torch

from . import ops

_LIB = "w8a8"


@torch.library.custom_op(f"{_LIB}::quant_act", mutates_args=())
def quant_act(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [rows, k] fp32 -> (int8 rows, scales [rows]) (llm/ref_model.py:191-196)."""
    return ops.quant_act(x)


@quant_act.register_fake
def _(x):
    return torch.empty(x.shape, dtype=torch.int8, device=x.device), x.new_empty(x.shape[0])


@torch.library.custom_op(f"{_LIB}::rmsnorm", mutates_args=())
def rmsnorm(x: torch.Tensor, g: torch.Tensor, eps: float) -> torch.Tensor:
    """(x * RSQRT(red_sum16(x * x) / n + eps)) * g per row (llm/ref_model.py:204-207)."""
    return ops.rmsnorm(x, g, eps)


@rmsnorm.register_fake
def _(x, g, eps):
    return torch.empty_like(x)


@torch.library.custom_op(f"{_LIB}::linear", mutates_args=())
def linear(xq: torch.Tensor, s_x: torch.Tensor, w: torch.Tensor, s_w: torch.Tensor) -> torch.Tensor:
    """(f32(xq . W^T) * s_w) * s_x on int8 rows, up to 16 of them (llm/ref_model.py:198-202)."""
    return ops.linear(xq, s_x, w, s_w)


@linear.register_fake
def _(xq, s_x, w, s_w):
    return xq.new_empty((xq.shape[0], w.shape[0]), dtype=torch.float32)


@torch.library.custom_op(f"{_LIB}::gemm", mutates_args=())
def gemm(xq: torch.Tensor, s_x: torch.Tensor, w: torch.Tensor, s_w: torch.Tensor) -> torch.Tensor:
    """The same linear for any row count on the tensor cores (tcgen05 kind::i8)."""
    return ops.gemm(xq, s_x, w, s_w)


@gemm.register_fake
def _(xq, s_x, w, s_w):
    return xq.new_empty((xq.shape[0], w.shape[0]), dtype=torch.float32)


@torch.library.custom_op(f"{_LIB}::linear_fused", mutates_args=())
def linear_fused(x: torch.Tensor, w: torch.Tensor, s_w: torch.Tensor, norm_g: torch.Tensor | None,
                 eps: float) -> torch.Tensor:
    """[rmsnorm ->] quant_act -> linear on fp32 rows (the decode GEMV with its fused prologue)."""
    return ops.linear_fused(x, w, s_w, norm_g=norm_g, eps=eps)


@linear_fused.register_fake
def _(x, w, s_w, norm_g, eps):
    return x.new_empty((x.shape[0], w.shape[0]))


@torch.library.custom_op(f"{_LIB}::ffn_swiglu", mutates_args=())
def ffn_swiglu(x: torch.Tensor, norm_g: torch.Tensor, eps: float, w_gate: torch.Tensor, s_gate: torch.Tensor,
               w_up: torch.Tensor, s_up: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Decode's fused SwiGLU dispatch: (h, int8 h, its scales) (llm/compile_model.py:295-328)."""
    scratch = ops.ffn_scratch(x.shape[0], x.device)
    h, hq, sh = ops.ffn_swiglu(x, norm_g, eps, w_gate, s_gate, w_up, s_up, scratch)
    return h, hq, sh


@ffn_swiglu.register_fake
def _(x, norm_g, eps, w_gate, s_gate, w_up, s_up):
    m, n = x.shape[0], w_gate.shape[0]
    return (x.new_empty((m, n)), torch.empty((m, n), dtype=torch.int8, device=x.device), x.new_empty(m))


@torch.library.custom_op(f"{_LIB}::embed", mutates_args=())
def embed(tokens: torch.Tensor, emb_q: torch.Tensor, emb_s: torch.Tensor) -> torch.Tensor:
    """f32(emb_q[token]) * emb_s[token] per token (llm/compile_model.py:192-201)."""
    return ops.embed(tokens, emb_q, emb_s)


@embed.register_fake
def _(tokens, emb_q, emb_s):
    return emb_s.new_empty((tokens.numel(), emb_q.shape[1]))


@torch.library.custom_op(f"{_LIB}::classifier", mutates_args=())
def classifier(x: torch.Tensor, w: torch.Tensor, s_w: torch.Tensor, norm_g: torch.Tensor, eps: float) -> torch.Tensor:
    """Final rmsnorm -> quant_act -> classifier GEMV (llm/compile_model.py:347-349)."""
    return ops.classifier(x, w, s_w, norm_g, eps)


@classifier.register_fake
def _(x, w, s_w, norm_g, eps):
    return x.new_empty((x.shape[0], w.shape[0]))


@torch.library.custom_op(f"{_LIB}::sfu", mutates_args=())
def sfu(func: int, x: torch.Tensor) -> torch.Tensor:
    """The overlay's table SFU elementwise: 0 EXP, 1 RECIP, 2 RSQRT, 3 SiLU, 4 GELU-tanh (llm/sfu.py)."""
    return ops.sfu(func, x)


@sfu.register_fake
def _(func, x):
    return torch.empty_like(x)


# ------------------------------------------------- block-scaled 8-bit KV cache
# (ops.KvBlocks as four tensors: codes int8 [slots, kv_heads, capacity, head_dim],
# scales fp32 [slots, kv_heads, capacity / block])
_KV = ("k_codes", "k_scale", "v_codes", "v_scale")


@torch.library.custom_op(f"{_LIB}::kvb_append", mutates_args=_KV)
def kvb_append(k: torch.Tensor, v: torch.Tensor, k_codes: torch.Tensor, k_scale: torch.Tensor, v_codes: torch.Tensor,
               v_scale: torch.Tensor, pos: torch.Tensor, start: torch.Tensor | None = None) -> None:
    """Rows k, v [rows, kv_heads, head_dim] into the cache (ops.kvb_append)."""
    ops.kvb_append(k, v, (k_codes, k_scale, v_codes, v_scale), pos, start)


@kvb_append.register_fake
def _(k, v, k_codes, k_scale, v_codes, v_scale, pos, start=None):
    return None


@torch.library.custom_op(f"{_LIB}::kvb_read", mutates_args=())
def kvb_read(k_codes: torch.Tensor, k_scale: torch.Tensor, v_codes: torch.Tensor, v_scale: torch.Tensor,
             pos: torch.Tensor, start: torch.Tensor, rows: int) -> tuple[torch.Tensor, torch.Tensor]:
    """The fp32 values held at the rows' positions (ops.kvb_read); rows behind
    the last sequence are zero."""
    k, v = (k_scale.new_zeros(rows, k_codes.shape[1], k_codes.shape[3]) for _ in range(2))
    return ops.kvb_read((k_codes, k_scale, v_codes, v_scale), pos, start, rows, k=k, v=v)


@kvb_read.register_fake
def _(k_codes, k_scale, v_codes, v_scale, pos, start, rows):
    shape = (rows, k_codes.shape[1], k_codes.shape[3])
    return k_scale.new_empty(shape), k_scale.new_empty(shape)


@torch.library.custom_op(f"{_LIB}::kvb_attn", mutates_args=("mass",))
def kvb_attn(q: torch.Tensor, k_codes: torch.Tensor, k_scale: torch.Tensor, v_codes: torch.Tensor,
             v_scale: torch.Tensor, pos: torch.Tensor, mass: torch.Tensor | None,
             scale: float | None = None) -> torch.Tensor:
    """Attention of one row per slot (ops.kvb_attn); mass or None."""
    return ops.kvb_attn(q, (k_codes, k_scale, v_codes, v_scale), pos, scale=scale, mass=mass)


@kvb_attn.register_fake
def _(q, k_codes, k_scale, v_codes, v_scale, pos, mass, scale=None):
    return q.new_empty(q.shape)


@torch.library.custom_op(f"{_LIB}::kvb_attn_rows", mutates_args=("mass",))
def kvb_attn_rows(q: torch.Tensor, k_codes: torch.Tensor, k_scale: torch.Tensor, v_codes: torch.Tensor,
                  v_scale: torch.Tensor, pos: torch.Tensor, start: torch.Tensor, mass: torch.Tensor | None,
                  scale: float | None = None) -> torch.Tensor:
    """Attention of prompt rows (ops.kvb_attn_rows), mass or None; rows behind
    the last sequence are zero."""
    return ops.kvb_attn_rows(q, (k_codes, k_scale, v_codes, v_scale), pos, start, scale=scale, mass=mass,
                             out=q.new_zeros(q.shape))


@kvb_attn_rows.register_fake
def _(q, k_codes, k_scale, v_codes, v_scale, pos, start, mass, scale=None):
    return q.new_empty(q.shape)


@torch.library.custom_op(f"{_LIB}::kvb_evict", mutates_args=_KV + ("mass",))
def kvb_evict(k_codes: torch.Tensor, k_scale: torch.Tensor, v_codes: torch.Tensor, v_scale: torch.Tensor,
              mass: torch.Tensor, count: torch.Tensor, keep: int, sink: int = 0,
              recent: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    """Every slot cut in place to its `keep` heaviest tokens (ops.kvb_evict)."""
    return ops.kvb_evict((k_codes, k_scale, v_codes, v_scale), mass, count, keep, sink=sink, recent=recent)


@kvb_evict.register_fake
def _(k_codes, k_scale, v_codes, v_scale, mass, count, keep, sink=0, recent=0):
    return count.new_empty((k_codes.shape[0], k_codes.shape[1], keep)), count.new_empty(k_codes.shape[0])


OPS = ("quant_act", "rmsnorm", "linear", "gemm", "linear_fused", "ffn_swiglu", "embed", "classifier", "sfu",
       "kvb_append", "kvb_read", "kvb_attn", "kvb_attn_rows", "kvb_evict")
