"""8-bit serving: quantised rows, integer products, and attention over a cache in 8 bits.

A row ``y`` stands as integers ``q = round(127 y / max|y|)`` (ties to even) and the scale ``max|y| / 127``: one scale for each
row of an activation, each output channel of a weight, each token and head of a cached key or value.  A row whose largest
value is below 2^-100 is stored as zeros with the scale 0; one that holds a NaN or an infinity as zeros with the scale NaN,
so that what is computed from it is NaN and not a number that looks like one.  Behind a norm the row is that of the whole formula;
its products of values and weights, in front of the norm's factor, and its sum of squares are fp32's: past its end they count as
infinities, and a row of products below 2^-120 as zeros.

A layer in 8 bits, with weights from ``quantize_rows(w)``::

    y, ys = rmsnorm_int8(x, norm_w, eps, residual=residual)
    qkv = linear_int8(y, ys, wqkv, wqkv_s)
    rope_kv_write_int8(qkv, positions, cos_sin, slots, cache, nq, nkv)
    a = paged_attention_int8(qkv, cache, meta, nq, nkv, scale)
    o = linear_int8(*quantize_rows(a), wo, wo_s)
    y, ys = rmsnorm_int8(o, post_w, eps, residual=residual)
    x = linear_int8(*silu_mul_int8(linear_int8(y, ys, wgu, wgu_s)), wdown, wdown_s)

Device tensors run on ``csrc/kernels/int8_*.hip``, on the current stream of their device; CPU tensors on the plain PyTorch
forms below.  There are no gradients: under grad mode, inputs that ask for one are refused, and so are those with a forward-mode
tangent.  On the device, calls inside ``torch.func`` transforms of their tensors and under ``torch.jit.trace`` or ``make_fx`` are
refused too, which would not see the launch.
"""
from __future__ import annotations

import math
import sys
from dataclasses import dataclass
from functools import lru_cache
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import attention as A
from ._lib import _dispatch_modes, _raw_stream, _tracing, _transforms, check, lib, ptr, scratch

HEAD_DIM = A.HEAD_DIM
TINY, LEAST = 2.0 ** -100, 2.0 ** -120
#: K of a product, at most: the sum of K products of 128 x 128 stays below 2^31
MAX_K = 131056
_ROW_TYPES = (torch.bfloat16, torch.float32)


_NO_GRADIENT = "the 8-bit operators have no gradients: detach the inputs or call under torch.no_grad()"
_grad_enabled = torch.is_grad_enabled
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _inputs(*tensors) -> int:
    """One device for all, whose number this is (-1: the CPU); none that asks for a gradient or that a launch by address would miss."""
    dev, grad = tensors[0].get_device(), _grad_enabled()
    for t in tensors:
        if t is not None:
            if t.get_device() != dev:
                raise ValueError(f"tensors on {tensors[0].device} and {t.device}")
            if grad and t.requires_grad:
                raise RuntimeError(_NO_GRADIENT)
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(_NO_GRADIENT)
    if dev >= 0 and (_tracing() is not None or _transforms() is not None or _dispatch_modes()):
        _seen(tensors)
    return dev


def _seen(tensors) -> None:
    """Refuses what records or rewrites torch's operators: it would have no part in a kernel launched by address."""
    if _tracing() is not None:
        raise RuntimeError("the 8-bit operators cannot be traced on the device: a trace would not hold the launch")
    if _transforms() is not None and any(torch._C._functorch.is_functorch_wrapped_tensor(t) for t in tensors if t is not None):
        raise RuntimeError("the 8-bit operators take no part in torch.func transforms on the device")
    fx = sys.modules.get("torch.fx.experimental.proxy_tensor")
    if fx is not None and fx.get_proxy_mode() is not None:
        raise RuntimeError("the 8-bit operators cannot be traced on the device: a trace would not hold the launch")


def _call(name: str, dev: int, *args) -> None:
    """The kernel's entry point on the current stream of device ``dev``, which is the current one meanwhile."""
    fn = getattr(lib(), name)
    if dev == _current_device():
        check(fn(*args, _stream(dev)), name)
    else:
        with torch.cuda.device(dev):
            check(fn(*args, _stream(dev)), name)


def _stream(dev: int) -> int:
    return _raw_stream(dev) if _raw_stream is not None else torch.cuda.current_stream(dev).cuda_stream


def _countable(*counts: int) -> None:
    """The kernels count rows and columns in 32 bits."""
    if max(counts) >= 1 << 31:
        raise ValueError(f"{max(counts)} rows or columns: at most 2^31 - 1 in one call")


def _pitch(t: torch.Tensor) -> int:
    """Values from row to row of a matrix whose rows are dense and start at multiples of 16 bytes; 0 of another."""
    (n, width), (ld, one) = t.shape, t.stride()
    if (one != 1 and width > 1) or t.data_ptr() & 15:
        return 0
    if n <= 1:
        return width
    return 0 if ld * t.element_size() & 15 else ld


def _apart(t: torch.Tensor) -> bool:
    """Whether the rows of a matrix that is written lie apart."""
    return t.shape[0] <= 1 or t.stride(0) >= t.shape[1]


def _quantised(y: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """The plain form on the last axis of an fp32 tensor (the quotient in 64 bits, so that ties are ties)."""
    top = y.abs().amax(-1, keepdim=True)
    fine = torch.isfinite(top)
    live = fine & (top >= TINY)
    q = torch.where(live, torch.round(127 * y.double() / torch.where(live, top, torch.ones_like(top)).double()), 0.0)
    scale = torch.where(live, top / 127.0, torch.where(fine, torch.zeros_like(top), torch.full_like(top, math.nan)))
    return q.to(torch.int8), scale.squeeze(-1)


# ------------------------------------------------------------------ rows
def _rows(mode: int, x: torch.Tensor, H: int, out, scale, w=None, residual=None, eps: float = 0.0):
    T = x.shape[0]
    dev, dtype = _inputs(x, out, scale, w, residual), x.dtype
    if dtype not in _ROW_TYPES:
        raise TypeError(f"rows must be bfloat16 or float32, not {dtype}")
    if H <= 0 or H % 16:
        raise ValueError(f"rows of a multiple of 16 values, not {H}")
    if out is None:
        out, ldq = torch.empty((T, H), dtype=torch.int8, device=x.device), H
    else:
        ldq = _pitch(out) if out.dtype == torch.int8 and out.shape == (T, H) and _apart(out) else 0
        if not ldq:
            raise ValueError(f"out must be int8 {[T, H]} with 16-byte rows that lie apart")
    if scale is None:
        scale = torch.empty(T, dtype=torch.float32, device=x.device)
    elif scale.dtype != torch.float32 or scale.shape != (T,) or not scale.is_contiguous():
        raise ValueError(f"scale must be contiguous float32 {[T]}")
    if w is not None and (w.dtype != dtype or w.shape != (H,)):
        raise ValueError(f"the norm's weight must be {dtype} {[H]}")
    if residual is not None and (residual.dtype != dtype or residual.shape != x.shape or not residual.is_contiguous()
                                 or residual.data_ptr() & 15):
        raise ValueError("the residual must be contiguous, 16-byte aligned and of the rows' shape and type")
    if dev >= 0:
        _countable(T)
        ld = _pitch(x)
        if not ld:
            x = x.clone(memory_format=torch.contiguous_format)
            ld = x.shape[1]
        if w is not None and not (w.is_contiguous() and w.data_ptr() & 15 == 0):
            w = w.clone(memory_format=torch.contiguous_format)
        _call("k8s_int8_rows", dev, mode, dtype is torch.float32, x.data_ptr(), ld, ptr(residual), ptr(w), out.data_ptr(), ldq,
              scale.data_ptr(), T, H, eps)
        return out, scale
    y = x.float()
    if mode == 1:
        g, u = y.split(H, dim=-1)
        y = g / (1 + torch.exp(-g)) * u
    elif mode == 2:
        if residual is not None:
            residual.copy_(y + residual.float())
            y = residual.float()
        top = (y * w.float()).abs().amax(-1, keepdim=True)
        ss = y.square().mean(-1, keepdim=True)
        y = y * torch.rsqrt(ss + eps) * w.float()
        y = y.masked_fill(top < LEAST, 0.0).masked_fill(~(torch.isfinite(top) & torch.isfinite(ss)), math.nan)
    q, s = _quantised(y)
    out.copy_(q)
    scale.copy_(s)
    return out, scale


def quantize_rows(x: torch.Tensor, out: Optional[torch.Tensor] = None,
                  scale: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``x`` [T, H] (bf16 or fp32) as int8 rows and fp32 scales [T].  Of a weight [N, K]: its output channels."""
    if x.dim() != 2:
        raise ValueError("rows must be a matrix")
    return _rows(0, x, x.shape[1], out, scale)


def silu_mul_int8(gu: torch.Tensor, out: Optional[torch.Tensor] = None,
                  scale: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``silu(gate) * up`` of ``gu`` [T, 2 I] (gate columns first), as ``norm.silu_mul``, in int8 rows: the product is
    quantised from fp32 and never written in a wider type."""
    if gu.dim() != 2 or gu.shape[1] % 2:
        raise ValueError("gate and up columns side by side in a matrix")
    return _rows(1, gu, gu.shape[1] // 2, out, scale)


def rmsnorm_int8(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: Optional[torch.Tensor] = None,
                 out: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``rmsnorm(x + residual) * weight`` in int8 rows; ``residual`` is updated in place to ``x + residual``, rounded to its
    type, and the norm is that of the rounded sum (as ``norm.rmsnorm``)."""
    if x.dim() != 2:
        raise ValueError("rows must be a matrix")
    return _rows(2, x, x.shape[1], out, scale, weight, residual, eps)


# ------------------------------------------------------------------ products
FEW, T32, T64, T64_128, T128_64, T128, T256, T128_256 = range(8)


@lru_cache(maxsize=4096)
def product_plan(M: int, N: int, K: int) -> Tuple[int, int, int]:
    """(kernel, runs of K, int32 numbers of workspace) of a product: the cheapest by the cost model beside the kernels."""
    p = lib().k8s_int8_gemm_plan(M, N, K)
    kind, runs = p & 255, p >> 8
    return kind, runs, lib().k8s_int8_gemm_part(M, N, kind, runs)


def linear_int8(x: torch.Tensor, x_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
                out_dtype: torch.dtype = torch.bfloat16, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``(x @ w.T) * x_scale[:, None] * w_scale (+ bias)`` for int8 ``x`` [M, K] and ``w`` [N, K], scales fp32 [M] and [N],
    ``bias`` fp32 [N]; bf16 or fp32 out.  The integer sum is exact, so a row's result does not depend on the rows beside it."""
    if x.dim() != 2 or w.dim() != 2 or x.shape[1] != w.shape[1]:
        raise ValueError(f"x [M, K] and w [N, K], not {list(x.shape)} and {list(w.shape)}")
    (M, K), N = x.shape, w.shape[0]
    dev = _inputs(x, x_scale, w, w_scale, bias, out)
    if x.dtype != torch.int8 or w.dtype != torch.int8:
        raise TypeError(f"x and w must be int8, not {x.dtype} and {w.dtype}")
    if not 0 < K <= MAX_K or K % 16:
        raise ValueError(f"K must be a multiple of 16 up to {MAX_K}, not {K}")
    for t, n in ((x_scale, M), (w_scale, N), (bias, N)):
        if t is not None and (t.dtype != torch.float32 or t.shape != (n,) or not t.is_contiguous()):
            raise ValueError(f"x_scale {[M]}, w_scale {[N]} and bias {[N]} must be contiguous float32, not {t.dtype} {list(t.shape)}")
    if out is None:
        if out_dtype not in _ROW_TYPES:
            raise TypeError(f"out_dtype must be bfloat16 or float32, not {out_dtype}")
        out, ldy = torch.empty((M, N), dtype=out_dtype, device=x.device), N
    else:
        if out.dtype not in _ROW_TYPES or out.shape != (M, N) or (out.stride(1) != 1 and N > 1) or not _apart(out):
            raise ValueError(f"out must be bfloat16 or float32 {[M, N]}, its rows dense and apart")
        ldy = out.stride(0) if M > 1 else N
    if M == 0 or N == 0:
        return out
    if dev >= 0:
        _countable(M, N)
        ldx, ldw = _pitch(x), _pitch(w)
        if not ldx:
            x = x.clone(memory_format=torch.contiguous_format)
            ldx = K
        if not ldw:
            raise ValueError("w's rows must be dense and start at multiples of 16 bytes")
        kind, runs, n = product_plan(M, N, K)
        part = torch.empty(n, dtype=torch.int32, device=x.device) if n else None
        _call("k8s_int8_gemm", dev, x.data_ptr(), ldx, x_scale.data_ptr(), w.data_ptr(), ldw, w_scale.data_ptr(), ptr(bias),
              out.data_ptr(), ldy, out.dtype is torch.float32, M, N, K, kind, runs, ptr(part), n)
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
        if _transforms() is not None and self.k.get_device() >= 0:
            _seen((self.k, self.v, self.k_scale, self.v_scale))
        NB, nkv, BS, D = self.k.shape
        if D != HEAD_DIM or self.v.shape != (NB, nkv, D, BS):
            raise ValueError("k must be [NB, nkv, BS, 128] and v [NB, nkv, 128, BS]")
        if BS <= 0 or BS % 64:
            raise ValueError(f"pages of a multiple of 64 tokens, not {BS}")
        if self.k.dtype != torch.int8 or self.v.dtype != torch.int8:
            raise ValueError("k and v must be int8")
        if any(s.dtype != torch.float32 or s.shape != (NB, nkv, BS) for s in (self.k_scale, self.v_scale)):
            raise ValueError("scales must be float32 [NB, nkv, BS]")
        if any(not t.is_contiguous() or t.data_ptr() % 16 or t.device != self.k.device for t in (self.k, self.v, self.k_scale, self.v_scale)):
            raise ValueError("the cache's tensors must be contiguous, 16-byte aligned and on one device")

    @staticmethod
    def empty(num_blocks: int, nkv: int, block_size: int, device) -> "Int8KV":
        """A pool of zeros (with scales of zero: a token that was never written is a zero)."""
        z = lambda *s, dtype: torch.zeros(*s, dtype=dtype, device=device)  # noqa: E731
        return Int8KV(z(num_blocks, nkv, block_size, HEAD_DIM, dtype=torch.int8), z(num_blocks, nkv, HEAD_DIM, block_size, dtype=torch.int8),
                      z(num_blocks, nkv, block_size, dtype=torch.float32), z(num_blocks, nkv, block_size, dtype=torch.float32))


def _heads(rows: torch.Tensor, cache: Int8KV, nq: int, nkv: int, width: int, what: str) -> None:
    if nkv <= 0 or nq <= 0 or nq % nkv:
        raise ValueError(f"{nq} query heads over {nkv} key heads")
    if cache.k.shape[1] != nkv:
        raise ValueError(f"a cache of {cache.k.shape[1]} heads, not {nkv}")
    if rows.dim() != 2 or rows.shape[1] < width:
        raise ValueError(f"{what} needs {width} columns")
    if rows.is_cuda and rows.dtype != torch.bfloat16:
        raise TypeError(f"{what} must be bfloat16, not {rows.dtype}")


def rope_kv_write_int8(qkv: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor, slots: Optional[torch.Tensor], cache: Int8KV,
                       nq: int, nkv: int) -> None:
    """Rotate the q heads of ``qkv`` [T, >= (nq + 2 nkv) 128] in place and write its keys (rotated, quantised from fp32) and
    values to the cache's slots.  The k and v columns stay as they came.  A row whose slot is negative (all rows, where
    ``slots`` is None) is rotated and not kept; nor is one whose slot the pool does not have.  A position outside ``cos_sin``
    takes its nearest row.  As in ``attention.rope_kv_write``, the rows of one call have different slots."""
    T = qkv.shape[0]
    _heads(qkv, cache, nq, nkv, (nq + 2 * nkv) * HEAD_DIM, "qkv")
    dev = _inputs(qkv, positions, cos_sin, slots, cache.k_scale, cache.v_scale)
    for t in (positions, slots):
        if t is not None and (t.dtype != torch.int32 or t.shape != (T,) or not t.is_contiguous()):
            raise ValueError(f"positions and slots must be contiguous int32 {[T]}, not {t.dtype} {list(t.shape)}")
    if cos_sin.dtype != torch.float32 or not cos_sin.is_contiguous() or cos_sin.dim() != 2 or cos_sin.shape[1] != HEAD_DIM or not cos_sin.shape[0]:
        raise ValueError("cos_sin must be contiguous float32 [positions, 128]")
    if not _apart(qkv):
        raise ValueError("the rows of qkv, which are written, must lie apart")
    NB, _, BS, D = cache.k.shape
    if T == 0:
        return
    if dev >= 0:
        ld = _pitch(qkv)
        if not ld or cos_sin.data_ptr() & 15:
            raise ValueError("the rows of qkv and cos_sin must be dense and start at multiples of 16 bytes")
        _call("k8s_int8_write", dev, qkv.data_ptr(), ld, positions.data_ptr(), cos_sin.data_ptr(), cos_sin.shape[0], ptr(slots),
              cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), T, nq, nkv, BS, NB * BS)
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
    ``attach_plan``): one plan serves both caches.  A plan for fewer heads, or whose lists or reply workspace are too short, is
    refused; a chunk's parts take a workspace of their own where the plan has none that holds them.  A row without a visible key
    gives zeros.  A context ends where its row of the table does; a page that the pool does not have counts as its nearest one."""
    T = q.shape[0]
    _heads(q, cache, nq, nkv, nq * HEAD_DIM, "q")
    NB, _, BS, D = cache.k.shape
    S, bt, ctx, starts = meta.num_seqs, meta.block_tables, meta.ctx_lens, meta.q_start
    dev = _inputs(q, bt, ctx, starts, cache.k_scale, cache.v_scale, out)
    if out is None:
        out, ldo = torch.empty((T, nq * D), dtype=q.dtype, device=q.device), nq * D
    else:
        if out.shape != (T, nq * D) or out.dtype != q.dtype or out.stride(1) != 1 or not _apart(out):
            raise ValueError("out must be [T, nq 128] of q's type, its rows dense and apart")
        ldo = out.stride(0) if T > 1 else nq * D
    if T == 0 or S == 0:
        return out
    if dev < 0:
        return _attention_plain(q, cache, meta, nq, nkv, scale, out)
    if bt.dtype != torch.int32 or bt.dim() != 2 or bt.shape[0] < S or bt.stride(1) != 1:
        raise ValueError("block_tables must be int32 [S, pages]")
    if S > 1 and bt.stride(0) < bt.shape[1]:
        raise ValueError("the rows of block_tables overlap")
    if _transforms() is not None:
        _seen(t for t in vars(meta).values() if isinstance(t, torch.Tensor))
    if ctx.dtype is not torch.int32 or starts.dtype is not torch.int32 or ctx.numel() < S or starts.numel() <= S or ctx.stride() != (1,) or starts.stride() != (1,):
        ctx, starts = _lengths(ctx, starts, S)
    ldq = _pitch(q)
    if not ldq:
        raise ValueError("q's rows must be dense and start at multiples of 16 bytes")
    G = nq // nkv
    common = (q.data_ptr(), ldq, cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), NB,
              bt.data_ptr(), bt.stride(0) if S > 1 else bt.shape[1], bt.shape[1], ctx.data_ptr(), starts.data_ptr())
    if meta.decode:
        if T != S:
            raise ValueError(f"a reply step has one row a sequence, not {T} for {S}")
        if G > 16:
            raise ValueError(f"{G} query heads a key head: a reply step takes 16")
        if meta.items is None:
            raise ValueError("the step has no plan: attach_decode_plan")
        _on(dev, meta.part_o, meta.part_ml)
        _listed(dev, 4 * meta.n_items, meta.items)
        n_items = meta.n_items
        if meta.d_n_items is not None:
            _listed(dev, 2, meta.d_n_items)
            n_items = meta.items.numel() // 4  # (the count that the device reads goes no further)
        if meta.item_tokens * G > 16:
            raise ValueError(f"a plan whose items have {meta.item_tokens} tokens, for fewer than {G} query heads a key head")
        if meta.n_parts > 1 and not _room(meta.part_o, meta.part_ml, S * nq * meta.n_parts):
            raise ValueError(f"a plan of several parts needs part_o and part_ml of {S} x {nq} x {meta.n_parts} rows")
        grid = max(1, meta.grid_waves or min(A.DECODE_WAVE_SLOTS, meta.n_items * nkv))
        _call("k8s_int8_attn_reply", dev, *common, S, nq, nkv, BS, scale, out.data_ptr(), ldo, ptr(meta.part_o), ptr(meta.part_ml),
              meta.n_parts, meta.part_size, meta.items.data_ptr(), n_items, ptr(meta.d_n_items), grid)
        return out
    rows = A.prefill_tile_tokens(G, BS) * G
    if rows > A.PF8_ROWS:
        raise ValueError(f"{G} query heads a key head: a tile takes {A.PF8_ROWS}")
    if meta.tile_seq is None or meta.tile_kv1 is None:
        raise ValueError("the step has no plan: attach_plan")
    _on(dev, meta.tile_seq, meta.pf_o, meta.pf_ml)
    part_o, part_ml, tiles, merged, own, runs = meta.pf_o, meta.pf_ml, meta.n_tiles, meta.n_merge, 0, 1
    if A.PF_ROWS % G or BS != 64:
        # Where heads or pages do not fit the bf16 cache's kernels the plan has tiles of about 64 rows over whole key ranges.  A workgroup
        # here takes 256 rows and finds them by itself.  Few of them cut their keys until there are as many as compute units, of
        # five pages each at least; from half as many on they make two rounds, which even out short and long tiles.  us by the plan's
        # tiles and by these, 10 + 2 x 2 heads: six threads' six tokens over 8064 keys 260 and 23, a prompt of 4096 225 and 101, two
        # of 513 27 and 26; 12 + 2 x 4: two chunks of 2000 over 2000 273 and 118, six prompts of 234 17.7 and 18.4.
        own = min(A.PF8_ROWS // G, T)
        tiles, merged, rows = T // own + S, 0, own * G
        blocks, pages = tiles * nkv, bt.shape[1] * BS // 64
        runs = max(1, min(256 // blocks, pages // 5) if blocks <= 128 else min(512 // blocks, pages // 16))
    else:
        if meta.tile_tokens * G > A.PF8_ROWS:
            raise ValueError(f"a plan whose tiles have {meta.tile_tokens} tokens, for fewer than {G} query heads a key head")
        _listed(dev, tiles, meta.tile_seq, meta.tile_tok0, meta.tile_len, meta.tile_kv0, meta.tile_kv1, meta.tile_slot)
        if merged:
            _listed(dev, merged, meta.m_tok0, meta.m_len, meta.m_slot0, meta.m_np)
    if merged or runs > 1:  # (a split tile's parts are tiles of the plan: no more than those, without a look at the device)
        rows_kept = (tiles * runs if own else meta.n_slots or tiles) * nkv * A.PF8_ROWS
        if own or not _room(part_o, part_ml, rows_kept):  # (none in the plan, or one for fewer key heads)
            part_o = scratch(rows_kept * D, torch.float32, q.device)
            part_ml = scratch(rows_kept * 2, torch.float32, q.device)
    _call("k8s_int8_attn_chunk", dev, *common, S, nq, nkv, BS, scale, out.data_ptr(), ldo, ptr(meta.tile_seq), ptr(meta.tile_tok0),
          ptr(meta.tile_len), ptr(meta.tile_kv0), ptr(meta.tile_kv1), ptr(meta.tile_slot), tiles, rows, ptr(meta.m_tok0),
          ptr(meta.m_len), ptr(meta.m_slot0), ptr(meta.m_np), merged, ptr(part_o), ptr(part_ml), A.PF8_ROWS, own, runs)
    return out


def _lengths(ctx: torch.Tensor, starts: torch.Tensor, S: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """ctx_lens and q_start as the kernels read them: one behind another (a column of a wider table is copied)."""
    if ctx.dtype != torch.int32 or starts.dtype != torch.int32 or ctx.dim() != 1 or starts.dim() != 1 or ctx.numel() < S or starts.numel() < S + 1:
        raise ValueError("ctx_lens must be int32 [S] and q_start int32 [S + 1]")
    return ctx.contiguous(), starts.contiguous()


def _room(part_o: Optional[torch.Tensor], part_ml: Optional[torch.Tensor], rows: int) -> bool:
    """Whether a plan's workspace holds the parts of so many rows: O, and its maximum and sum."""
    return (part_o is not None and part_ml is not None and part_o.dtype is torch.float32 and part_ml.dtype is torch.float32
            and part_o.numel() >= HEAD_DIM * rows and part_ml.numel() >= 2 * rows and part_o.is_contiguous() and part_ml.is_contiguous())


def _on(dev: int, *tensors) -> None:
    for t in tensors:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"a plan on {t.device} for device {dev}")


def _listed(dev: int, n: int, *lists) -> None:
    """A plan's lists: what the kernels read of them is there, one behind another."""
    for t in lists:
        if t is None:
            raise ValueError("a list of the step's plan is missing")
        if t.dtype is not torch.int32 or t.numel() < n or not t.is_contiguous():
            raise ValueError(f"a plan's list must be contiguous int32 of {n}, not {t.dtype} {list(t.shape)}")
        if t.get_device() != dev:
            raise ValueError(f"a plan on {t.device} for device {dev}")


def _attention_plain(q, cache: Int8KV, meta: A.AttnMeta, nq, nkv, scale, out):
    starts, ctx = meta.q_start.tolist(), meta.ctx_lens.tolist()
    BS, D, G = cache.k.shape[2], HEAD_DIM, nq // nkv
    for s in range(meta.num_seqs):
        n, c = starts[s + 1] - starts[s], min(max(0, ctx[s]), meta.block_tables.shape[1] * BS)
        at = meta.block_tables[s, :-(-c // BS)].long().clamp(0, cache.k.shape[0] - 1)
        k = (cache.k[at].float() * cache.k_scale[at][..., None]).permute(1, 0, 2, 3).reshape(nkv, -1, D)[:, :c]
        v = (cache.v[at].float() * cache.v_scale[at][:, :, None]).permute(1, 0, 3, 2).reshape(nkv, -1, D)[:, :c]
        # a value's scale that is no number makes its key's score none, so that rows that do not see the key stay as they are
        odd = ~torch.isfinite(cache.v_scale[at].permute(1, 0, 2).reshape(nkv, 1, 1, -1)[..., :c])
        v = v.masked_fill(odd[:, 0, 0, :, None], 0.0)
        rows = q[starts[s]:starts[s] + n, :nq * D].float().view(n, nkv, G, D).permute(1, 2, 0, 3)
        x = torch.matmul(rows, k[:, None].transpose(-1, -2)) * scale
        hidden = torch.arange(c) > (ctx[s] - n + torch.arange(n))[:, None]
        x = x.masked_fill(odd, math.nan).masked_fill(hidden, -math.inf)
        p = torch.softmax(x, -1).masked_fill(hidden, 0.0)  # (a row without a key: zeros)
        o = torch.matmul(p, v[:, None]) if c else torch.zeros(nkv, G, n, D)
        out[starts[s]:starts[s] + n] = o.permute(2, 0, 1, 3).reshape(n, nq * D).to(out.dtype)
    return out
