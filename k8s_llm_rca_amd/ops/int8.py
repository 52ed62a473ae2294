"""8-bit serving: quantised rows, integer products, and attention over a cache in 8 bits.

A row ``y`` stands as integers ``q = round(127 y / max|y|)`` (ties to even) and the scale ``max|y| / 127``: one scale for each
row of an activation, each output channel of a weight, each token and head of a cached key or value.  A row whose largest
value is below 2^-100 is stored as zeros with the scale 0; one that holds a NaN or an infinity as zeros with the scale NaN,
so that what is computed from it is NaN and not a number that looks like one.

A layer in 8 bits, with weights from ``quantize_rows(w)``::

    y, ys = rmsnorm_int8(x, norm_w, eps, residual=residual)
    qkv = linear_int8(y, ys, wqkv, wqkv_s)
    rope_kv_write_int8(qkv, positions, cos_sin, slots, cache, nq, nkv)
    a = paged_attention_int8(qkv, cache, meta, nq, nkv, scale)
    o = linear_int8(*quantize_rows(a), wo, wo_s)
    y, ys = rmsnorm_int8(o, post_w, eps, residual=residual)
    x = linear_int8(*silu_mul_int8(linear_int8(y, ys, wgu, wgu_s)), wdown, wdown_s)

Device tensors run on ``csrc/kernels/int8_*.hip``, on the current stream of their device; CPU tensors on the plain PyTorch
forms below.  There are no gradients: under grad mode, inputs that ask for one are refused.
"""
from __future__ import annotations

import math
from contextlib import nullcontext
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import attention as A
from ._lib import check, lib, ptr, stream_ptr, use_hip

HEAD_DIM = A.HEAD_DIM
TINY = 2.0 ** -100
#: K of a product, at most: the sum of K products of 128 x 128 stays below 2^31
MAX_K = 131056
_ROW_TYPES = (torch.bfloat16, torch.float32)


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _inputs(*tensors) -> None:
    """One device for all; none that asks for a gradient."""
    dev = tensors[0].device
    for t in tensors:
        if t is None:
            continue
        _need(t.device == dev, f"tensors on {dev} and {t.device}")
        if t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("the 8-bit operators have no gradients: detach the inputs or call under torch.no_grad()")


def _on(t: torch.Tensor):
    """The tensor's device as the current one while a kernel is launched."""
    return nullcontext() if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)


def _aligned(t: torch.Tensor) -> bool:
    """Rows one behind another, each starting at a multiple of 16 bytes."""
    return t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and (t.shape[0] <= 1 or t.stride(0) * t.element_size() % 16 == 0)


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _quantised(y: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """The plain form on the last axis of an fp32 tensor."""
    top = y.abs().amax(-1, keepdim=True)
    fine = torch.isfinite(top)
    live = fine & (top >= TINY)
    q = torch.where(live, torch.round(y * (127.0 / torch.where(live, top, torch.ones_like(top)))), torch.zeros_like(y))
    scale = torch.where(live, top / 127.0, torch.where(fine, torch.zeros_like(top), torch.full_like(top, math.nan)))
    return q.to(torch.int8), scale.squeeze(-1)


# ------------------------------------------------------------------ rows
def _rows(mode: int, x: torch.Tensor, H: int, out, scale, w=None, residual=None, eps: float = 0.0):
    T = x.shape[0]
    _inputs(x, out, scale, w, residual)
    if x.dtype not in _ROW_TYPES:
        raise TypeError(f"rows must be bfloat16 or float32, not {x.dtype}")
    _need(H > 0 and H % 16 == 0, f"rows of a multiple of 16 values, not {H}")
    if out is None:
        out = torch.empty((T, H), dtype=torch.int8, device=x.device)
    if scale is None:
        scale = torch.empty(T, dtype=torch.float32, device=x.device)
    _need(out.dtype == torch.int8 and out.shape == (T, H) and _aligned(out), "out must be int8 [T, H] with 16-byte rows")
    _need(scale.dtype == torch.float32 and scale.shape == (T,) and scale.is_contiguous(), "scale must be contiguous float32 [T]")
    if w is not None:
        _need(w.dtype == x.dtype and w.shape == (H,), f"the norm's weight must be {x.dtype} [{H}]")
    if residual is not None:
        _need(residual.dtype == x.dtype and residual.shape == x.shape and residual.is_contiguous() and residual.data_ptr() % 16 == 0,
              "the residual must be contiguous, 16-byte aligned and of the rows' shape and type")
    if use_hip(x):
        if not _aligned(x):
            x = x.clone(memory_format=torch.contiguous_format)
        if w is not None and not (w.is_contiguous() and w.data_ptr() % 16 == 0):
            w = w.clone(memory_format=torch.contiguous_format)
        with _on(x):
            check(lib().k8s_int8_rows(mode, int(x.dtype == torch.float32), ptr(x), _ld(x), ptr(residual), ptr(w), ptr(out), _ld(out),
                                      ptr(scale), T, H, float(eps), stream_ptr(x)), "int8_rows")
        return out, scale
    y = x.float()
    if mode == 1:
        g, u = y.split(H, dim=-1)
        y = g / (1 + torch.exp(-g)) * u
    elif mode == 2:
        if residual is not None:
            residual.copy_(y + residual.float())
            y = residual.float()
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) * w.float()
    q, s = _quantised(y)
    out.copy_(q)
    scale.copy_(s)
    return out, scale


def quantize_rows(x: torch.Tensor, out: Optional[torch.Tensor] = None,
                  scale: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``x`` [T, H] (bf16 or fp32) as int8 rows and fp32 scales [T].  Of a weight [N, K]: its output channels."""
    _need(x.dim() == 2, "rows must be a matrix")
    return _rows(0, x, x.shape[1], out, scale)


def silu_mul_int8(gu: torch.Tensor, out: Optional[torch.Tensor] = None,
                  scale: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``silu(gate) * up`` of ``gu`` [T, 2 I] (gate columns first), as ``norm.silu_mul``, in int8 rows: the product is
    quantised from fp32 and never written in a wider type."""
    _need(gu.dim() == 2 and gu.shape[1] % 2 == 0, "gate and up columns side by side in a matrix")
    return _rows(1, gu, gu.shape[1] // 2, out, scale)


def rmsnorm_int8(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: Optional[torch.Tensor] = None,
                 out: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``rmsnorm(x + residual) * weight`` in int8 rows; ``residual`` is updated in place to ``x + residual``, rounded to its
    type, and the norm is that of the rounded sum (as ``norm.rmsnorm``)."""
    _need(x.dim() == 2, "rows must be a matrix")
    return _rows(2, x, x.shape[1], out, scale, weight, residual, eps)


# ------------------------------------------------------------------ products
def linear_int8(x: torch.Tensor, x_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
                out_dtype: torch.dtype = torch.bfloat16, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``(x @ w.T) * x_scale[:, None] * w_scale (+ bias)`` for int8 ``x`` [M, K] and ``w`` [N, K], scales fp32 [M] and [N],
    ``bias`` fp32 [N]; bf16 or fp32 out.  The integer sum is exact, so a row's result does not depend on the rows beside it."""
    _need(x.dim() == 2 and w.dim() == 2 and x.shape[1] == w.shape[1], "x [M, K] and w [N, K]")
    M, K = x.shape
    N = w.shape[0]
    _inputs(x, x_scale, w, w_scale, bias, out)
    if x.dtype != torch.int8 or w.dtype != torch.int8:
        raise TypeError(f"x and w must be int8, not {x.dtype} and {w.dtype}")
    _need(0 < K <= MAX_K and K % 16 == 0, f"K must be a multiple of 16 up to {MAX_K}, not {K}")
    for t, n, name in ((x_scale, M, "x_scale"), (w_scale, N, "w_scale"), (bias, N, "bias")):
        _need(t is None or (t.dtype == torch.float32 and t.shape == (n,) and t.is_contiguous()), f"{name} must be contiguous float32 [{n}]")
    if out is None:
        if out_dtype not in _ROW_TYPES:
            raise TypeError(f"out_dtype must be bfloat16 or float32, not {out_dtype}")
        out = torch.empty((M, N), dtype=out_dtype, device=x.device)
    _need(out.dtype in _ROW_TYPES and out.shape == (M, N) and out.stride(1) == 1, "out must be bfloat16 or float32 [M, N], its rows dense")
    if M == 0 or N == 0:
        return out
    if use_hip(x):
        if not _aligned(x):
            x = x.clone(memory_format=torch.contiguous_format)
        _need(_aligned(w), "w's rows must be dense and start at multiples of 16 bytes")
        with _on(x):
            check(lib().k8s_int8_gemm(ptr(x), _ld(x), ptr(x_scale), ptr(w), _ld(w), ptr(w_scale), ptr(bias), ptr(out), _ld(out),
                                      int(out.dtype == torch.float32), M, N, K, stream_ptr(x)), "int8_gemm")
        return out
    # (in fp64 every partial sum is an integer below 2^53: exact)
    y = (x.double() @ w.double().T).float() * x_scale[:, None] * w_scale
    out.copy_(y if bias is None else y + bias)
    return out


# ------------------------------------------------------------------ the cache
@dataclass
class Int8KV:
    """One layer's paged keys and values in 8 bits: ``k`` [NB, nkv, BS, 128] and ``v`` [NB, nkv, 128, BS] (transposed
    pages, as the bf16 cache has them) int8, ``k_scale`` and ``v_scale`` [NB, nkv, BS] fp32.  264 bytes a token and head, of
    the bf16 cache's 512."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    def __post_init__(self):
        NB, nkv, BS, D = self.k.shape
        _need(D == HEAD_DIM and self.v.shape == (NB, nkv, D, BS), "k must be [NB, nkv, BS, 128] and v [NB, nkv, 128, BS]")
        _need(BS > 0 and BS % 64 == 0, f"pages of a multiple of 64 tokens, not {BS}")
        _need(self.k.dtype == torch.int8 == self.v.dtype, "k and v must be int8")
        for s in (self.k_scale, self.v_scale):
            _need(s.dtype == torch.float32 and s.shape == (NB, nkv, BS), "scales must be float32 [NB, nkv, BS]")
        for t in (self.k, self.v, self.k_scale, self.v_scale):
            _need(t.is_contiguous() and t.data_ptr() % 16 == 0 and t.device == self.k.device,
                  "the cache's tensors must be contiguous, 16-byte aligned and on one device")

    @staticmethod
    def empty(num_blocks: int, nkv: int, block_size: int, device) -> "Int8KV":
        """A pool of zeros (with scales of zero: a token that was never written is a zero)."""
        z = lambda *s, dtype: torch.zeros(*s, dtype=dtype, device=device)  # noqa: E731
        return Int8KV(z(num_blocks, nkv, block_size, HEAD_DIM, dtype=torch.int8), z(num_blocks, nkv, HEAD_DIM, block_size, dtype=torch.int8),
                      z(num_blocks, nkv, block_size, dtype=torch.float32), z(num_blocks, nkv, block_size, dtype=torch.float32))


def _heads(rows: torch.Tensor, cache: Int8KV, nq: int, nkv: int, width: int, what: str) -> None:
    _inputs(rows, cache.k)
    _need(nkv > 0 and nq > 0 and nq % nkv == 0, f"{nq} query heads over {nkv} key heads")
    _need(cache.k.shape[1] == nkv, f"a cache of {cache.k.shape[1]} heads, not {nkv}")
    _need(rows.dim() == 2 and rows.shape[1] >= width, f"{what} needs {width} columns")
    if rows.is_cuda and rows.dtype != torch.bfloat16:
        raise TypeError(f"{what} must be bfloat16, not {rows.dtype}")


def _ints(*tensors) -> None:
    for t, shape, name in tensors:
        _need(t.dtype == torch.int32 and t.is_contiguous() and t.shape == shape, f"{name} must be contiguous int32 {list(shape)}")


def rope_kv_write_int8(qkv: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor, slots: Optional[torch.Tensor], cache: Int8KV,
                       nq: int, nkv: int) -> None:
    """Rotate the q heads of ``qkv`` [T, >= (nq + 2 nkv) 128] in place and write its keys (rotated, quantised from fp32) and
    values to the cache's slots.  The k and v columns stay as they came.  A row whose slot is negative (all rows, where
    ``slots`` is None) is rotated and not kept; nor is one whose slot the pool does not have.  As in
    ``attention.rope_kv_write``, the rows of one call have different slots."""
    T = qkv.shape[0]
    _heads(qkv, cache, nq, nkv, (nq + 2 * nkv) * HEAD_DIM, "qkv")
    _inputs(qkv, positions, cos_sin, slots)
    _ints((positions, (T,), "positions"), *([] if slots is None else [(slots, (T,), "slots")]))
    _need(cos_sin.dtype == torch.float32 and cos_sin.is_contiguous() and cos_sin.dim() == 2 and cos_sin.shape[1] == HEAD_DIM
          and cos_sin.shape[0] > 0, "cos_sin must be contiguous float32 [positions, 128]")
    NB, _, BS, D = cache.k.shape
    if T == 0:
        return
    if use_hip(qkv):
        _need(_aligned(qkv) and cos_sin.data_ptr() % 16 == 0, "qkv's rows must be dense and start at multiples of 16 bytes")
        with _on(qkv):
            check(lib().k8s_int8_write(ptr(qkv), _ld(qkv), ptr(positions), ptr(cos_sin), cos_sin.shape[0], ptr(slots), ptr(cache.k),
                                       ptr(cache.v), ptr(cache.k_scale), ptr(cache.v_scale), T, nq, nkv, BS, NB * BS, stream_ptr(qkv)),
                  "int8_write")
        return
    nh = nq + nkv
    cos, sin = cos_sin[positions.long().clamp(0, cos_sin.shape[0] - 1)][:, None].chunk(2, -1)
    x = qkv[:, :(nq + 2 * nkv) * D].float().view(T, -1, D)
    a, b = x[:, :nh].chunk(2, -1)
    turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    qkv[:, :nq * D] = turned[:, :nq].reshape(T, -1).to(qkv.dtype)
    if slots is None:
        return
    kept = (slots >= 0) & (slots < NB * BS)
    at = slots.long()[kept]
    page, off = at // BS, at % BS
    k, ks = _quantised(turned[kept][:, nq:])
    v, vs = _quantised(x[kept][:, nh:])
    cache.k[page, :, off], cache.k_scale[page, :, off] = k, ks
    cache.v[page, :, :, off], cache.v_scale[page, :, off] = v, vs


def paged_attention_int8(q: torch.Tensor, cache: Int8KV, meta: A.AttnMeta, nq: int, nkv: int, scale: float,
                         out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of ``q`` [T, >= nq 128] (row stride free) over the 8-bit pages -> [T, nq 128], for reply tokens and
    chunks alike.  ``meta`` is the step's, with the plan that ``attention.paged_attention`` takes (``attach_decode_plan`` or
    ``attach_plan``): one plan serves both caches.  A row without a visible key gives zeros."""
    T = q.shape[0]
    _heads(q, cache, nq, nkv, nq * HEAD_DIM, "q")
    NB, _, BS, D = cache.k.shape
    S = meta.num_seqs
    _inputs(q, meta.block_tables, meta.ctx_lens, meta.q_start, out)
    if out is None:
        out = torch.empty((T, nq * D), dtype=q.dtype, device=q.device)
    _need(out.shape == (T, nq * D) and out.dtype == q.dtype and out.stride(1) == 1, "out must be [T, nq 128] of q's type, its rows dense")
    if T == 0 or S == 0:
        return out
    if not use_hip(q):
        return _attention_plain(q, cache, meta, nq, nkv, scale, out)
    bt = meta.block_tables
    _need(bt.dtype == torch.int32 and bt.dim() == 2 and bt.shape[0] >= S and bt.stride(1) == 1, "block_tables must be int32 [S, pages]")
    _need(meta.ctx_lens.dtype == torch.int32 == meta.q_start.dtype and meta.ctx_lens.numel() >= S and meta.q_start.numel() >= S + 1,
          "ctx_lens must be int32 [S] and q_start int32 [S + 1]")
    _need(_aligned(q), "q's rows must be dense and start at multiples of 16 bytes")
    G, L = nq // nkv, lib()
    common = (ptr(q), _ld(q), ptr(cache.k), ptr(cache.v), ptr(cache.k_scale), ptr(cache.v_scale), NB, ptr(bt), bt.stride(0) if S > 1 else bt.shape[1],
              ptr(meta.ctx_lens), ptr(meta.q_start))
    if meta.decode:
        _need(T == S, "a reply step has one row a sequence")
        _need(G <= 16, f"{G} query heads a key head: a reply step takes 16")
        _need(meta.items is not None and meta.items.dtype == torch.int32, "the step has no plan: attach_decode_plan")
        _need(meta.n_parts == 1 or meta.part_o is not None, "a plan of several parts needs part_o and part_ml")
        grid = max(1, meta.grid_waves or min(A.DECODE_WAVE_SLOTS, meta.n_items * nkv))
        with _on(q):
            check(L.k8s_int8_attn_reply(*common, S, nq, nkv, BS, float(scale), ptr(out), _ld(out), ptr(meta.part_o), ptr(meta.part_ml),
                                        meta.n_parts, meta.part_size, ptr(meta.items), meta.n_items, ptr(meta.d_n_items), grid,
                                        stream_ptr(q)), "int8_attn_reply")
        return out
    rows = A.prefill_tile_tokens(G, BS) * G
    _need(rows <= A.PF8_ROWS, f"{G} query heads a key head: a tile takes {A.PF8_ROWS}")
    _need(meta.tile_seq is not None and meta.tile_kv1 is not None, "the step has no plan: attach_plan")
    if meta.n_merge and meta.pf_o is None:
        meta.pf_o, meta.pf_ml = A.prefill_workspace(nkv, q.device, max(meta.m_slot0_end(), 1))
    with _on(q):
        check(L.k8s_int8_attn_chunk(*common, nq, nkv, BS, float(scale), ptr(out), _ld(out), ptr(meta.tile_seq), ptr(meta.tile_tok0),
                                    ptr(meta.tile_len), ptr(meta.tile_kv0), ptr(meta.tile_kv1), ptr(meta.tile_slot), meta.n_tiles, rows,
                                    ptr(meta.m_tok0), ptr(meta.m_len), ptr(meta.m_slot0), ptr(meta.m_np), meta.n_merge, ptr(meta.pf_o),
                                    ptr(meta.pf_ml), A.PF8_ROWS, stream_ptr(q)), "int8_attn_chunk")
    return out


def _attention_plain(q, cache: Int8KV, meta: A.AttnMeta, nq, nkv, scale, out):
    starts, ctx = meta.q_start.tolist(), meta.ctx_lens.tolist()
    BS, D, G = cache.k.shape[2], HEAD_DIM, nq // nkv
    for s in range(meta.num_seqs):
        n, c = starts[s + 1] - starts[s], max(0, ctx[s])
        at = meta.block_tables[s, :-(-c // BS)].long()
        k = (cache.k[at].float() * cache.k_scale[at][..., None]).permute(1, 0, 2, 3).reshape(nkv, -1, D)[:, :c]
        v = (cache.v[at].float() * cache.v_scale[at][:, :, None]).permute(1, 0, 3, 2).reshape(nkv, -1, D)[:, :c]
        rows = q[starts[s]:starts[s] + n, :nq * D].float().view(n, nkv, G, D).permute(1, 2, 0, 3)
        x = torch.matmul(rows, k[:, None].transpose(-1, -2)) * scale
        hidden = torch.arange(c) > (c - n + torch.arange(n))[:, None]
        x = x.masked_fill(hidden, -math.inf)
        p = torch.softmax(x, -1).masked_fill(hidden, 0.0)  # (a row without a key: zeros)
        o = torch.matmul(p, v[:, None]) if c else torch.zeros(nkv, G, n, D)
        out[starts[s]:starts[s] + n] = o.permute(2, 0, 1, 3).reshape(n, nq * D).to(out.dtype)
    return out
