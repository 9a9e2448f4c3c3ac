"""Public op API used by the models.

Every op takes flattened token tensors (``[T, ...]`` with ``T = B * S``). On CUDA tensors the op
runs the sm_100a kernels through hand-written autograd Functions (``ops.cuda_fns``), which
accumulate weight gradients straight into each parameter's fp32 ``main_grad``; if the compiled
extension is missing this raises. On CPU tensors the op evaluates the fp32 oracle
(``ops.reference``) under torch autograd -- the same definitions the kernels are tested against.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch
import torch.nn.functional as F

from . import reference as R
from .layout import split_gate_up
from .quant import dequantize_w4, quantize_w4  # noqa: F401  (public names of the 4-bit weights)


_CUDA = None


def _cuda():
    """``cuda_fns``, which needs the built extension; kept, as an import statement costs 0.6 us a call."""
    global _CUDA
    if _CUDA is None:
        from . import cuda_fns

        _CUDA = cuda_fns
    return _CUDA


# ---------------------------------------------------------------------------------- embedding


def embed(ids: torch.Tensor, table: torch.Tensor) -> torch.Tensor:
    if ids.is_cuda:
        return _cuda().embed(ids, table)
    return F.embedding(ids, table)


def linear(x: torch.Tensor, w: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ w^T`` (+ residual)."""
    if x.is_cuda:
        return _cuda().linear(x, w, residual)
    y = x @ w.t().to(x.dtype)
    return y if residual is None else residual + y


# ------------------------------------------------------------------------------ norms


def rms_gated_norm(x, w_rms, eps: float, w_down=None, w_up=None):
    """RMSNorm followed (optionally) by GatedNorm (megagpt-speedrun/model.py:288-328)."""
    if x.is_cuda:
        return _cuda().rms_gated_norm(x, w_rms, eps, w_down, w_up)
    y = R.rms_norm(x, w_rms, eps)
    if w_down is not None:
        y = R.gated_norm(y, w_down, w_up)
    return y


def rms_gated_norm_res(x, w_rms, eps: float, w_down=None, w_up=None):
    """``(norm(x), residual)``: the normalised input and the tensor to use as the block's residual
    stream (on CUDA an alias of ``x`` whose gradient is summed inside the norm's backward kernel)."""
    if x.is_cuda:
        return _cuda().rms_gated_norm(x, w_rms, eps, w_down, w_up, passthrough=True)
    return rms_gated_norm(x, w_rms, eps, w_down, w_up), x


# -------------------------------------------------------------------------------- attention


class AttnShape:
    """Static description of one attention call."""

    def __init__(self, batch, seq, heads, kv_heads, head_dim, window=0, qk_mult=1.0, qk_norm=True,
                 xsa=True, head_gate=True, rope_theta=10000.0, llama3=None):
        self.batch, self.seq, self.heads, self.kv_heads, self.head_dim = batch, seq, heads, kv_heads, head_dim
        self.window, self.qk_mult, self.qk_norm = window, qk_mult, qk_norm
        self.xsa, self.head_gate = xsa, head_gate
        self.rope_theta, self.llama3 = rope_theta, llama3

    @property
    def q_cols(self):
        return self.heads * self.head_dim

    @property
    def kv_cols(self):
        return self.kv_heads * self.head_dim


_ROPE_CACHE: dict = {}


def rope_tables(seq, head_dim, theta, device, llama3=None):
    key = (seq, head_dim, theta, str(device), None if llama3 is None else tuple(sorted(llama3.items())))
    t = _ROPE_CACHE.get(key)
    if t is None:
        t = R.rope_cos_sin(seq, head_dim, theta, device=device, llama3=llama3)
        _ROPE_CACHE[key] = t
    return t


def attention_block(h, x, w_qkv, attn_gate, w_o, shape: AttnShape, segment_ids=None):
    """``x + W_o( gate * XSA( attn( rope(qknorm(W_q h)), rope(qknorm(W_k h)), W_v h ) ) )``
    (megagpt-speedrun/model.py:255-285). ``h`` is the normalised block input, ``x`` the residual."""
    if h.is_cuda:
        return _cuda().attention_block(h, x, w_qkv, attn_gate, w_o, shape, segment_ids)
    b, s, nh, hkv, hd = shape.batch, shape.seq, shape.heads, shape.kv_heads, shape.head_dim
    qkv = h @ w_qkv.t()
    q = qkv[:, : shape.q_cols].reshape(b, s, nh, hd)
    k = qkv[:, shape.q_cols: shape.q_cols + shape.kv_cols].reshape(b, s, hkv, hd)
    v = qkv[:, shape.q_cols + shape.kv_cols:].reshape(b, s, hkv, hd)
    if shape.qk_norm:
        q = R.rms_norm_noparam(q)
        k = R.rms_norm_noparam(k)
    cos, sin = rope_tables(s, hd, shape.rope_theta, h.device, shape.llama3)
    q = R.apply_rope(q, cos, sin)
    k = R.apply_rope(k, cos, sin)
    q = q * shape.qk_mult
    seg = None if segment_ids is None else segment_ids.view(b, s)
    o = R.attention(q, k, v, window=shape.window, segment_ids=seg)
    if shape.xsa or shape.head_gate:
        gate_w = attn_gate if attn_gate is not None else torch.zeros(nh, h.shape[1], device=h.device)
        o = R.xsa_head_gate(o, v, h.view(b, s, -1), gate_w, xsa=shape.xsa, head_gate=shape.head_gate)
    o = o.reshape(b * s, nh * hd)
    return x + o @ w_o.t()


# -------------------------------------------------------------------------------------- MLPs


def dense_mlp(h, w_in, w_down, *, glu: bool, act: str, residual=None):
    """Dense MLP: SwiGLU (blocked gate/up rows in ``w_in``) or plain ``act(h W_in^T) W_down^T``."""
    if h.is_cuda:
        return _cuda().dense_mlp(h, w_in, w_down, glu, act, residual)
    z = h @ w_in.t()
    if glu:
        g, u = split_gate_up(z, w_down.shape[1])
        a = R.activation(g, act) * u
    else:
        a = R.activation(z, act)
    y = a @ w_down.t()
    return y if residual is None else residual + y


# ------------------------------------------------------------------------------------ router


class RouterOut:
    """Routing decision and the differentiable router losses of one MoE layer."""

    def __init__(self, selected, combine, keep, z_loss, lbl, sparsity, counts, entropy, beta, expected, realized):
        self.selected, self.combine, self.keep = selected, combine, keep
        self.z_loss, self.lbl, self.sparsity = z_loss, lbl, sparsity
        self.counts, self.entropy, self.beta = counts, entropy, beta
        self.expected_active, self.realized_active = expected, realized


def route(h, w_router, router_bias, k: int, *, adaptive=False, threshold=None, k_min=0, temp=1.0,
          qb_count: int = 1, need_beta: bool = True, logit_bias=None):
    """Router of megagpt-speedrun/model.py:559-634: fp32 logits, top-(K+1) on biased logits,
    sigmoid combine weights on unbiased logits, per-layer z-loss / LBL / sparsity penalty and the
    local QB beta (the cross-rank mean is taken by the caller). ``logit_bias`` ``[E]`` is an optional
    learned additive logit bias (depth-conditioned routing), differentiated like the logits."""
    if h.is_cuda:
        return _cuda().route(h, w_router, router_bias, k, adaptive, threshold, k_min, temp, qb_count, need_beta,
                             logit_bias)
    out = R.route(h, w_router, router_bias, k, adaptive=adaptive, threshold=threshold, k_min=k_min, temp=temp,
                  logit_bias=logit_bias)
    e = w_router.shape[0]
    st = R.routing_stats(out["selected"], out["probs"], out["logits"], e, k)
    beta = R.qb_beta(out["logits"].detach(), out["alpha"].detach(), qb_count) if need_beta else None
    sparsity = out["expected_active"].mean() / e
    return RouterOut(out["selected"], out["combine"], out["hard_keep"], st["router_z_loss"],
                     st["load_balancing_loss"], sparsity, st["routing_counts"], st["routing_entropy"], beta,
                     out["expected_active"].mean() / e, out["realized_active"].mean() / e)


def moe_experts(h, r: RouterOut, w_gate_up, w_down, *, capacity: int | None, act: str = "silu", residual=None):
    """Routed expert SwiGLU MLP over the capacity layout (``capacity=None``: dropless)."""
    if h.is_cuda:
        return _cuda().moe_experts(h, r, w_gate_up, w_down, capacity, act, residual)
    from .layout import blocked_rows_to_gate_up

    g, u = blocked_rows_to_gate_up(w_gate_up)
    w_std = torch.cat([g, u], dim=1)
    keep = r.keep if not bool(r.keep.all()) else None
    y = R.moe_experts(h, r.selected, r.combine, w_std, w_down, capacity=capacity, keep=keep, act=act)
    return y if residual is None else residual + y


def capacity_for(tokens: int, k: int, experts: int, factor: float, align: int = 128) -> int:
    """Per-expert buffer rows: ceil(factor * tokens * k / experts) rounded up to ``align``."""
    c = int(math.ceil(factor * tokens * k / experts))
    return max(align, (c + align - 1) // align * align)


# ------------------------------------------------------------------------------------- loss


def cross_entropy(h, w_out, labels, weights, *, z_weight: float = 0.0):
    """Fused linear + softmax cross-entropy with z-loss; weighted mean over tokens."""
    if h.is_cuda:
        return _cuda().cross_entropy(h, w_out, labels, weights, z_weight)
    return R.fused_linear_cross_entropy(h, w_out, labels, weights, z_weight=z_weight)


def ngram_embed(ids: torch.Tensor, table: torch.Tensor, orders, n_hash: int) -> torch.Tensor:
    """Hashed n-gram input embedding ``[B*S, rank]`` (mean over orders x hashes)."""
    if ids.is_cuda:
        return _cuda().ngram_embed(ids, table, orders, n_hash)
    return R.ngram_embed(ids, table, orders, n_hash)


# ------------------------------------------------------------------------ quantised serving path
#
# A paged KV cache in 8 bits, its block tables, and products with 4-bit weights. None of them has a
# backward pass; the ones that take activations refuse inputs that require a gradient.


def _serving_only(name: str, *tensors) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{name} has no backward pass")


class BlockPlan(NamedTuple):
    """One step of a paged cache (all int32). Rows behind the last new token have slot and request
    -1 and position 0. ``status`` is 0, or has the bits 1 (too few free pages), 2 (a request outgrows
    its row of the table), 4 (more new tokens than rows), 8 (a negative length or a bad free count):
    then nothing was placed, the tables are unchanged and ``lens`` / ``free_count`` are the old ones."""

    lens: torch.Tensor        # [R] lengths with the new tokens
    free_count: torch.Tensor  # [1] free pages left
    starts: torch.Tensor      # [R + 1] first row of each request's new tokens
    slots: torch.Tensor       # [rows] page * page_size + offset of each new token
    requests: torch.Tensor    # [rows] its request
    positions: torch.Tensor   # [rows] its position in the request
    status: torch.Tensor      # [1]


def block_tables_extend(tables, lens, new_lens, free_pages, free_count, page_size: int, rows: int) -> BlockPlan:
    """Give ``new_lens [R]`` further tokens of each request their pages and rows, on the device.

    ``tables [R, width]`` (request r's pages, in order; written in place), ``lens [R]`` (tokens that
    are cached), ``free_pages`` (a stack of unused pages: the first ``free_count [1]`` entries, taken
    from the end), all int32. ``rows`` is the number of rows of the step (the new tokens of all
    requests, packed, and padding). Only ``tables`` changes, so calling it again gives the same plan;
    the caller keeps the plan's ``lens`` and ``free_count`` when it takes the step. Up to 4096
    requests."""
    if tables.is_cuda:
        return BlockPlan._make(_cuda().ext().block_tables_extend(tables, lens, new_lens, free_pages, free_count,
                                                                 page_size, rows))
    return BlockPlan(*R.block_tables_extend(tables, lens, new_lens, free_pages, free_count, page_size, rows))


def block_tables_release(tables, lens, done, free_pages, free_count, page_size: int) -> torch.Tensor:
    """Push the pages of the requests marked in ``done [R]`` (bool) onto the free stack and empty
    them (``lens`` 0, table entries -1), in place. Returns a status ``[1]`` like ``BlockPlan``'s; if
    it is not 0 nothing changed."""
    if tables.is_cuda:
        return _cuda().ext().block_tables_release(tables, lens, done, free_pages, free_count, page_size)
    return R.block_tables_release(tables, lens, done, free_pages, free_count, page_size)


def kv8_append(k, v, k_cache, v_cache, k_scale, v_scale, slots) -> None:
    """Write rows of keys and values (``[rows, kv_heads, head_dim]`` bf16, head_dim 64 or 128) to
    their slots of a cache of e4m3 codes ``[pages, kv_heads, page, head_dim]`` (page 32, 64 or 128)
    with fp32 scales ``[pages, kv_heads]``, in place. Keys and values have caches and scales of their own.

    Scales are powers of two. A row at offset 0 starts its page anew; rows further on keep the page's
    scale or raise it, and raising it rescales the codes before them. Values that are not finite are
    stored as NaN, and a page that holds such a value (not a key) gets a negative ``v_scale``. Rows
    with a slot outside the cache (the padding's -1) are skipped. The rows of one page must be
    consecutive rows, each with the slot that follows the last one's, as a ``BlockPlan`` gives them, and
    a page must belong to one request: two runs of rows in one page (a gap between their slots makes
    two) would race for its scale."""
    _serving_only("kv8_append", k, v)
    if k.is_cuda:
        _cuda().ext().kv8_append(k, v, k_cache, v_cache, k_scale, v_scale, slots)
    else:
        R.kv8_append(k, v, k_cache, v_cache, k_scale, v_scale, slots)


def kv8_attention(q, k_cache, v_cache, k_scale, v_scale, tables, lens, *, starts=None, scale: float | None = None,
                  out=None) -> torch.Tensor:
    """Causal attention of the requests' newest rows over their cached tokens (GQA), ``[rows, heads,
    head_dim]`` bf16.

    ``lens [R]`` counts the cached tokens with the new ones, which are already appended. Rows
    ``starts[r] .. starts[r + 1]`` of ``q`` are the last tokens of request r; without ``starts`` each
    request has one row. A row that sees no token is zero. A row that sees a page outside the cache is
    NaN, and so is every other row of a request that is longer than its table. Rows of no request (before ``starts[0]``, behind
    ``starts[R]``) are left as they were in ``out`` (which overlaps no input), and are zero without it. ``starts`` must ascend
    within ``0 .. rows``; with others nothing is computed. The cache is one that ``kv8_append`` wrote:
    scales are powers of two, and a page of values with NaN codes has a negative one.

    Scores, softmax sums and outputs are summed in fp32; the weights meet the values rounded to f16
    (2^-12 of a weight), well inside the result's own rounding to bf16."""
    _serving_only("kv8_attention", q)
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    if q.is_cuda:
        return _cuda().ext().kv8_attention(q, k_cache, v_cache, k_scale, v_scale, tables, lens, starts, scale, out)
    return R.kv8_attention(q, k_cache, v_cache, k_scale, v_scale, tables, lens, starts, scale, out)


def linear_w4(x, codes, scales, *, residual=None, glu: bool = False) -> torch.Tensor:
    """``x [T, K] @ w^T`` with the 4-bit weights of ``quantize_w4`` (+ ``residual [T, N]``), bf16.

    ``glu``: the weight holds block-interleaved gate and up rows (``ops.layout``) and the result is
    ``silu(gate) * up`` ``[T, N / 2]``. Up to 64 rows the weights stay in 4 bits on their way to the
    tensor cores (rows of ``x`` start at multiples of 16 bytes); more rows run the dense GEMM on
    weights written out in bf16 (each rounded once more, and a temporary of ``2 N K`` bytes, which
    takes longer than the GEMM on bf16 weights: it is for prompts of a model that has only these).
    The residual is added in fp32, before the one rounding of the result; with ``glu`` above 64 rows gate
    and up are rounded to bf16 before the activation, as in ``dense_mlp``."""
    _serving_only("linear_w4", x, residual)
    if not x.is_cuda:
        return R.linear_w4(x, codes, scales, residual, glu)
    if x.shape[0] <= 64:
        fns = _cuda()
        return fns.ext().linear_w4(x, codes, scales, residual, glu, fns.err_flag(x.device) if x.shape[0] > 32 else None)
    return _cuda().linear_w4_dense(x, codes, scales, residual, glu)
