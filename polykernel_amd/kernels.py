"""Torch-tensor front end of the gfx950 kernels.

Function names and argument meaning follow the reference's golden interface
(tests/golden/golden.py:48-172, tests/golden/quant_golden.py:71-101): bf16 in,
bf16 out, fused ops equal to their compositions.  Tensors are device tensors
(torch is only the allocator and stream provider); every call goes through the
C-ABI of libpolykernel_amd.so on torch's current stream.  A failing launch
raises PolyKernelError with the library's message.
"""
from __future__ import annotations

import math
import struct
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import check

bf16 = torch.bfloat16


# torch's own handle of the current stream: torch.cuda.current_stream() builds a
# Stream object around it, 2.8 us of the 9.3 us that a small call took.
_current_device = getattr(torch._C, "_cuda_getDevice", None)
_current_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream() -> int:
    if _current_raw_stream is None or _current_device is None:
        return torch.cuda.current_stream().cuda_stream
    return _current_raw_stream(_current_device())


def _dev(t: torch.Tensor, dtype: torch.dtype, name: str) -> int:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name}: tensor must live on a GPU (got {t.device})")
    if t.dtype != dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: tensor must be contiguous")
    return t.data_ptr()


def _opt(t: Optional[torch.Tensor], dtype, name) -> Optional[int]:
    return None if t is None else _dev(t, dtype, name)


def rmsnorm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """golden.rmsnorm (golden.py:83-90) via launch_rmsnorm."""
    cols = x.shape[-1]
    rows = x.numel() // cols if cols else 0
    out = torch.empty_like(x)
    check(_lib.load().launch_rmsnorm(_dev(x, bf16, "x"), _opt(weight, bf16, "weight"),
                                     _dev(out, bf16, "out"), rows, cols, eps, _stream()),
          "launch_rmsnorm")
    return out


def fused_residual_rmsnorm(x: torch.Tensor, residual: torch.Tensor,
                           weight: Optional[torch.Tensor] = None, eps: float = 1e-5,
                           config: Optional[dict] = None) -> torch.Tensor:
    """golden.fused_residual_rmsnorm (golden.py:108-112); `config` picks one of
    pk_op_configs("fused_residual_rmsnorm", rows, cols, 0) (tuning/test hook
    pk_fused_residual_rmsnorm_config)."""
    if x.shape != residual.shape:
        raise ValueError("x and residual must have the same shape")
    cols = x.shape[-1]
    rows = x.numel() // cols
    out = torch.empty_like(x)
    args = (_dev(x, bf16, "x"), _dev(residual, bf16, "residual"), _opt(weight, bf16, "weight"),
            _dev(out, bf16, "out"), rows, cols, eps)
    if config is None:
        check(_lib.load().launch_fused_residual_rmsnorm(*args, _stream()), "launch_fused_residual_rmsnorm")
    else:
        check(_lib.load().pk_fused_residual_rmsnorm_config(*args, _lib.Config(**config), _stream()),
              "pk_fused_residual_rmsnorm_config")
    return out


def gelu(x: torch.Tensor) -> torch.Tensor:
    """golden.gelu (golden.py:63-66); bit-exact with kernels/cpu launch_gelu_cpu."""
    out = torch.empty_like(x)
    check(_lib.load().launch_gelu(_dev(x, bf16, "x"), _dev(out, bf16, "out"), x.numel(), _stream()),
          "launch_gelu")
    return out


def softmax(x: torch.Tensor) -> torch.Tensor:
    """golden.softmax over the last axis (golden.py:75-80)."""
    cols = x.shape[-1]
    out = torch.empty_like(x)
    check(_lib.load().launch_softmax(_dev(x, bf16, "x"), _dev(out, bf16, "out"),
                                     x.numel() // cols, cols, _stream()), "launch_softmax")
    return out


def fused_softmax_mask(logits: torch.Tensor, mask: torch.Tensor, config: Optional[dict] = None) -> torch.Tensor:
    """golden.fused_softmax_mask (golden.py:115-117) on fp32 logits + bf16 additive mask;
    `config` picks one of pk_op_configs("fused_softmax_mask", rows, cols, 0)
    (tuning/test hook pk_fused_softmax_mask_config)."""
    if logits.shape != mask.shape:
        raise ValueError("logits and mask must have the same shape")
    cols = logits.shape[-1]
    out = torch.empty(logits.shape, dtype=bf16, device=logits.device)
    args = (_dev(logits, torch.float32, "logits"), _dev(mask, bf16, "mask"), _dev(out, bf16, "out"),
            logits.numel() // cols, cols)
    if config is None:
        check(_lib.load().launch_fused_softmax_mask(*args, _stream()), "launch_fused_softmax_mask")
    else:
        check(_lib.load().pk_fused_softmax_mask_config(*args, _lib.Config(**config), _stream()),
              "pk_fused_softmax_mask_config")
    return out


def _mk(a: torch.Tensor, b: torch.Tensor) -> Tuple[int, int, int]:
    K = a.shape[-1]
    if b.dim() != 2 or b.shape[0] != K:
        raise ValueError(f"contraction mismatch: a[..., {K}] @ b{tuple(b.shape)}")
    return a.numel() // K, b.shape[1], K


def matmul(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """golden.matmul (golden.py:58-60): [..., M, K] @ [K, N]."""
    M, N, K = _mk(a, b)
    out = torch.empty(*a.shape[:-1], N, dtype=bf16, device=a.device)
    check(_lib.load().launch_matmul(_dev(a, bf16, "a"), _dev(b, bf16, "b"), _dev(out, bf16, "out"),
                                    M, N, K, _stream()), "launch_matmul")
    return out


def gemm_ex(epi: int, a, b, bias=None, residual=None, tile: int = -1) -> torch.Tensor:
    """Explicit-tile GEMM (tuning/test hook pk_gemm_ex)."""
    M, N, K = _mk(a, b)
    out = torch.empty(*a.shape[:-1], N, dtype=bf16, device=a.device)
    check(_lib.load().pk_gemm_ex(epi, _dev(a, bf16, "a"), _dev(b, bf16, "b"), _dev(out, bf16, "out"),
                                 _opt(bias, bf16, "bias"), _opt(residual, bf16, "residual"),
                                 M, N, K, tile, _stream()), "pk_gemm_ex")
    return out


def fused_rmsnorm_matmul(x: torch.Tensor, w: torch.Tensor, weight: Optional[torch.Tensor] = None,
                         eps: float = 1e-5) -> torch.Tensor:
    """golden.fused_rmsnorm_matmul (golden.py:96-100); `weight` is the rmsnorm gamma."""
    M, N, K = _mk(x, w)
    out = torch.empty(*x.shape[:-1], N, dtype=bf16, device=x.device)
    lib = _lib.load()
    if weight is None:
        rc = lib.launch_fused_rmsnorm_matmul(_dev(x, bf16, "x"), _dev(w, bf16, "w"),
                                             _dev(out, bf16, "out"), M, N, K, eps, _stream())
        check(rc, "launch_fused_rmsnorm_matmul")
    else:
        rc = lib.launch_fused_rmsnorm_matmul_gamma(_dev(x, bf16, "x"), _dev(weight, bf16, "weight"),
                                                   _dev(w, bf16, "w"), _dev(out, bf16, "out"),
                                                   M, N, K, eps, _stream())
        check(rc, "launch_fused_rmsnorm_matmul_gamma")
    return out


def fused_matmul_bias_gelu(x: torch.Tensor, w: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """golden.fused_matmul_bias_gelu (golden.py:103-105)."""
    M, N, K = _mk(x, w)
    out = torch.empty(*x.shape[:-1], N, dtype=bf16, device=x.device)
    check(_lib.load().launch_fused_matmul_bias_gelu(_dev(x, bf16, "x"), _dev(w, bf16, "w"),
                                                    _dev(b, bf16, "b"), _dev(out, bf16, "out"),
                                                    M, N, K, _stream()),
          "launch_fused_matmul_bias_gelu")
    return out


def fused_matmul_bias_residual(x: torch.Tensor, w: torch.Tensor, b: Optional[torch.Tensor],
                               residual: torch.Tensor) -> torch.Tensor:
    """add(bias(matmul(x, w), b), residual) -- the MLP down-projection epilogue."""
    M, N, K = _mk(x, w)
    out = torch.empty(*x.shape[:-1], N, dtype=bf16, device=x.device)
    check(_lib.load().launch_fused_matmul_bias_residual(
        _dev(x, bf16, "x"), _dev(w, bf16, "w"), _opt(b, bf16, "b"), _dev(residual, bf16, "residual"),
        _dev(out, bf16, "out"), M, N, K, _stream()), "launch_fused_matmul_bias_residual")
    return out


def mlp_block(x, gamma, w1, b1, w2, b2, eps: float = 1e-6, workspace: Optional[torch.Tensor] = None):
    """RMSNorm -> MatMul W1 + b1 -> GELU -> MatMul W2 + b2 -> + x (config-2 block)."""
    M, d = x.numel() // x.shape[-1], x.shape[-1]
    F = w1.shape[1]
    lib = _lib.load()
    need = lib.pk_mlp_block_workspace_size(M, d, F)
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
    out = torch.empty_like(x)
    check(lib.launch_mlp_block(_dev(x, bf16, "x"), _opt(gamma, bf16, "gamma"), _dev(w1, bf16, "w1"),
                               _dev(b1, bf16, "b1"), _dev(w2, bf16, "w2"), _dev(b2, bf16, "b2"),
                               _dev(out, bf16, "out"), M, d, F, eps, workspace.data_ptr(),
                               workspace.numel(), _stream()), "launch_mlp_block")
    return out


def kv_cache_update(cache: torch.Tensor, new: torch.Tensor) -> torch.Tensor:
    """Out-of-place KV append: concat(cache, new) on axis 2 (attention.cpp:63-92)."""
    B, H, Sc, D = cache.shape
    Sn = new.shape[2]
    out = torch.empty(B, H, Sc + Sn, D, dtype=bf16, device=cache.device)
    check(_lib.load().launch_kv_cache_update(_dev(cache, bf16, "cache"), _dev(new, bf16, "new"),
                                             _dev(out, bf16, "out"), B, H, Sc, Sn, D, _stream()),
          "launch_kv_cache_update")
    return out


def attention_prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                      scale: Optional[float] = None, causal: bool = True) -> torch.Tensor:
    """SDPA over the full key set (attention.cpp:95-163)."""
    B, H, Sq, D = q.shape
    Skv = k.shape[2]
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    out = torch.empty_like(q)
    check(_lib.load().launch_attention_prefill(_dev(q, bf16, "q"), _dev(k, bf16, "k"), _dev(v, bf16, "v"),
                                               _dev(out, bf16, "out"), B, H, Sq, Skv, D, scale,
                                               int(causal), _stream()), "launch_attention_prefill")
    return out


def fused_kv_append_attention(q, k_new, v_new, k_cache, v_cache, s_cache: int,
                              scale: Optional[float] = None, causal: bool = True) -> torch.Tensor:
    """In-place append of k_new/v_new at row s_cache of the caches, then attention
    over the s_cache + S_q keys (golden.fused_kv_append_attention, golden.py:139-172)."""
    B, H, Sq, D = q.shape
    cap = k_cache.shape[2]
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    out = torch.empty_like(q)
    check(_lib.load().launch_fused_kv_append_attention(
        _dev(q, bf16, "q"), _dev(k_cache, bf16, "k_cache"), _dev(v_cache, bf16, "v_cache"),
        _dev(k_new, bf16, "k_new"), _dev(v_new, bf16, "v_new"), _dev(out, bf16, "out"),
        B, H, Sq, s_cache, D, cap, scale, int(causal), _stream()), "launch_fused_kv_append_attention")
    return out


# ---- serving from a paged cache (no counterpart in the reference) ----------------
def rotary_frequencies(dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0, low: float = 1.0,
                       high: float = 4.0, original: int = 0, device="cuda") -> Tuple[torch.Tensor, float]:
    """(turns, magnitude) for `rotary` and `paged_kv_append`: the revolutions per
    position of each of dim / 2 pairs, in fp64 on `device`, with the frequencies
    stretched for long contexts as `scaling` says ("none", "linear", "base",
    "bands", "ramp"; include/polykernel_amd.h, pk_rotary_frequencies)."""
    if scaling not in _lib.ROTARY_SCALINGS:
        raise ValueError(f"scaling: one of {_lib.ROTARY_SCALINGS}, got {scaling!r}")
    turns = torch.empty(max(dim // 2, 0), dtype=torch.float64)
    mag = _lib.D()
    check(_lib.load().pk_rotary_frequencies(dim, base, _lib.ROTARY_SCALINGS.index(scaling), factor, low, high, original,
                                            turns.data_ptr() or None, mag), "pk_rotary_frequencies")
    return turns.to(device), mag.value


def _device() -> int:
    if _current_device is None or not torch.cuda.is_initialized():
        return torch.cuda.current_device() if torch.cuda.is_available() else -2
    return _current_device()


def _elsewhere(t: torch.Tensor, name: str, dev: int) -> Exception:
    if not t.is_cuda:
        return ValueError(f"{name}: tensor must live on a GPU (got {t.device})")
    return ValueError(f"{name}: tensor is on {t.device}, the current device is cuda:{dev}")


def _heads(t: torch.Tensor, dims: int, name: str, dev: int) -> Tuple[int, ...]:
    """The strides of a bf16 tensor of heads on device `dev`: any, with head dims contiguous."""
    if isinstance(t, torch.Tensor) and t.dtype is bf16 and t.get_device() == dev:
        strides = t.stride()
        if len(strides) == dims and (strides[-1] == 1 or t.shape[-1] <= 1):
            return strides
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor")
    if t.dtype != bf16:
        raise TypeError(f"{name}: expected {bf16}, got {t.dtype}")
    if t.dim() != dims:
        raise ValueError(f"{name}: expected {dims} dimensions, got shape {tuple(t.shape)}")
    if t.get_device() != dev:
        raise _elsewhere(t, name, dev)
    raise ValueError(f"{name}: the head dim must be contiguous (strides {t.stride()})")


def _table(t: torch.Tensor, shape, dtype: torch.dtype, name: str, dev: int) -> int:
    """A contiguous table of the given shape on device `dev`."""
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.get_device() == dev and t.is_contiguous():
        return t.data_ptr()
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor")
    if t.dtype != dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.get_device() != dev:
        raise _elsewhere(t, name, dev)
    raise ValueError(f"{name}: tensor must be contiguous")


_INT = 0x7FFFFFFF  # numbers that the C entry points take in 32 bits (ctypes would cut larger ones)


# a result's memory: 1.6 us where torch.empty with a shape, type and device takes 3.7
def _result(like: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(like, memory_format=torch.contiguous_format)


def _rotation(turns: torch.Tensor, interleaved: bool, inverse: bool, magnitude: float, dev: int) -> bytes:
    n = turns.numel() if isinstance(turns, torch.Tensor) else 0
    return _lib.Rotary.pack(_table(turns, (n,), torch.float64, "turns", dev), 2 * n, interleaved, inverse, magnitude)


def rotary(x: torch.Tensor, positions: torch.Tensor, turns: torch.Tensor, *, interleaved: bool = False,
           magnitude: float = 1.0, inverse: bool = False, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotate the first 2 len(turns) dims of every head by its position: pairs (i, i + len(turns)),
    or (2 i, 2 i + 1) when `interleaved`, by positions * turns[i] revolutions, times `magnitude`.

    x is [tokens, heads, D] with positions [tokens], or [B, heads, S, D] with positions [S] or
    [B, S] (int32); any strides with contiguous head dims.  `inverse` rotates back, which is the
    gradient: dx = rotary(dy, positions, turns, inverse=True) with the same magnitude.  `out` (contiguous by default) may
    be `x`."""
    if not isinstance(x, torch.Tensor) or x.dim() not in (3, 4):
        raise ValueError("x: expected a tensor [tokens, heads, D] or [B, heads, S, D]")
    dev, dims = _device(), x.dim()
    xs = _heads(x, dims, "x", dev)
    if out is None:
        out = _result(x)
        os_ = out.stride()
    else:
        os_ = _heads(out, dims, "out", dev)
        if out.shape != x.shape:
            raise ValueError(f"out: expected shape {tuple(x.shape)}, got {tuple(out.shape)}")
    if dims == 3:
        S, H, D = x.shape
        B, per = 1, 0
        xs, os_ = (0, xs[0], xs[1]), (0, os_[0], os_[1])
        pos = _table(positions, (S,), torch.int32, "positions", dev)
    else:
        B, H, S, D = x.shape
        xs, os_ = (xs[0], xs[2], xs[1]), (os_[0], os_[2], os_[1])
        whole = isinstance(positions, torch.Tensor) and positions.dim() == 2
        per = S if whole else 0
        pos = _table(positions, (B, S) if whole else (S,), torch.int32, "positions", dev)
    if B * S > _INT or H * D > _INT:
        raise ValueError(f"x: {B * S} tokens of {H * D} elements (each at most {_INT})")
    rot = _rotation(turns, interleaved, inverse, magnitude, dev)
    check(_lib.load().launch_rotary(x.data_ptr(), _strides3(*xs), out.data_ptr(), _strides3(*os_), pos, per, B, S, H, D,
                                    rot, _stream()), "launch_rotary")
    return out


_strides3 = struct.Struct("qqq").pack


def _tokens(t: torch.Tensor, name: str, heads: int, dim: int, tokens: int, dev: int) -> bytes:
    """A [tokens, heads, dim] tensor (heads 0: any number)."""
    try:
        (token, head, last), (n, h, d) = t.stride(), t.shape
        fine = t.dtype is bf16 and t.get_device() == dev and (last == 1 or d <= 1)
    except (AttributeError, ValueError):
        fine = False
    if not fine:
        _heads(t, 3, name, dev)  # says what is wrong
    if n != tokens or d != dim or (heads and h != heads):
        raise ValueError(f"{name}: expected [{tokens}, {heads or 'heads'}, {dim}], got {tuple(t.shape)}")
    if n > _INT or h > _INT:
        raise ValueError(f"{name}: {n} tokens of {h} heads (each at most {_INT})")
    return _lib.Tokens.pack(t.data_ptr(), token, head)


def _refuse_paged(k_cache, v_cache, page_table, kv_len, dev: int) -> None:
    """Says what is wrong with the tables or caches of a paged call."""
    _heads(k_cache, 4, "k_cache", dev), _heads(v_cache, 4, "v_cache", dev)
    if k_cache.shape != v_cache.shape:
        raise ValueError("k_cache and v_cache must have the same shape, got "
                         f"{tuple(k_cache.shape)}, {tuple(v_cache.shape)}")
    if not isinstance(kv_len, torch.Tensor) or kv_len.dim() != 1:
        raise ValueError("kv_len: expected an int32 tensor [sequences]")
    B = kv_len.shape[0]
    _table(kv_len, (B,), torch.int32, "kv_len", dev)
    if not isinstance(page_table, torch.Tensor) or page_table.dim() != 2 or page_table.shape[0] != B:
        raise ValueError(f"page_table: expected an int32 tensor [{B}, pages of a sequence]")
    if page_table.dtype != torch.int32:
        raise TypeError(f"page_table: expected {torch.int32}, got {page_table.dtype}")
    if page_table.get_device() != dev:
        raise _elsewhere(page_table, "page_table", dev)
    raise ValueError("page_table: the pages of a sequence must be contiguous")


def _paged(k_cache, v_cache, page_table, q_start, kv_len, tokens: int, max_q: int, max_kv: int, dev: int):
    """(cache, heads, dim, batch) for the C entry points, once everything is as it has to be: one
    condition, since a step's call takes no longer than its checks."""
    try:
        (k0, k1, k2, k3), (v0, v1, v2, v3) = k_cache.stride(), v_cache.stride()
        pages, heads, rows, dim = shape = k_cache.shape
        B, width = page_table.shape
        t0, t1 = page_table.stride()
        fine = (shape == v_cache.shape and ((k3 == 1 and v3 == 1) or dim <= 1) and (t1 == 1 or width <= 1)
                and k_cache.dtype is bf16 and v_cache.dtype is bf16 and page_table.dtype is kv_len.dtype is torch.int32
                and kv_len.shape == (B,) and kv_len.is_contiguous()
                and k_cache.get_device() == v_cache.get_device() == page_table.get_device() == kv_len.get_device() == dev)
    except (AttributeError, ValueError):
        fine = False
    if not fine:
        _refuse_paged(k_cache, v_cache, page_table, kv_len, dev)
    if pages > _INT:
        raise ValueError(f"k_cache: {pages} pages (at most {_INT})")
    if q_start is not None:
        q_start = _table(q_start, (B + 1,), torch.int32, "q_start", dev)
    elif tokens != B:
        raise ValueError(f"q_start: without it every sequence has one token (got {tokens} tokens, {B} sequences)")
    return (_lib.PagedCache.pack(k_cache.data_ptr(), v_cache.data_ptr(), k0, k1, k2, v0, v1, v2, pages, rows, heads, dim), heads,
            dim, _lib.PagedBatch.pack(page_table.data_ptr(), t0, width, q_start or 0, kv_len.data_ptr(), B, tokens, max_q, max_kv))


def paged_kv_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    page_table: torch.Tensor, q_start: Optional[torch.Tensor], kv_len: torch.Tensor, *,
                    q: Optional[torch.Tensor] = None, turns: Optional[torch.Tensor] = None, interleaved: bool = False,
                    magnitude: float = 1.0, q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Write the new tokens' keys and values into their pages, the keys (and q, which is returned)
    rotated by their positions on the way where `turns` is given (as in `rotary`).

    k and v [tokens, heads, D] and q [tokens, q heads, D] hold the sequences' new tokens one
    sequence behind the other: q_start[b] to q_start[b + 1] (int32 [sequences + 1]; None: one token
    each).  kv_len[b] (int32) counts the sequence's keys with the new ones; the key at position p
    goes to row p % page_size of page page_table[b, p // page_size] of the caches
    [pages, heads, page_size, D].  Strides are free as long as head dims are contiguous.  Tokens
    behind the last sequence's, and tokens on a page number outside the cache, write nothing.
    `q_out` may be `q`."""
    T, dev = k.shape[0] if isinstance(k, torch.Tensor) and k.dim() == 3 else 0, _device()
    cache, heads, D, batch = _paged(k_cache, v_cache, page_table, q_start, kv_len, T, 0, 0, dev)
    kt, vt = _tokens(k, "k", heads, D, T, dev), _tokens(v, "v", heads, D, T, dev)
    rot = None if turns is None else _rotation(turns, interleaved, False, magnitude, dev)
    qt = ot = None
    Hq = 0
    if q is not None:
        if rot is None:
            raise ValueError("q: without turns there is nothing to do for the queries")
        qt = _tokens(q, "q", 0, D, T, dev)
        Hq = q.shape[1]
        if q_out is None:
            q_out = _result(q)
            ot = _lib.Tokens.pack(q_out.data_ptr(), Hq * D, D)
        else:
            ot = _tokens(q_out, "q_out", Hq, D, T, dev)
    elif q_out is not None:
        raise ValueError("q_out: there is no q")
    check(_lib.load().launch_paged_kv_append(kt, vt, qt, ot, Hq, cache, batch, rot, _stream()), "launch_paged_kv_append")
    return q_out


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                    q_start: Optional[torch.Tensor], kv_len: torch.Tensor, *, max_q: Optional[int] = None, max_kv: int = 0,
                    scale: Optional[float] = None, causal: bool = True, window: int = 0,
                    workspace: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the new tokens q [tokens, q heads, D] over the pages of their sequences
    (arguments as `paged_kv_append`, which comes first).  Query head h reads key head
    h // (q heads / heads).  A token at position p sees the keys up to p (causal) or all kv_len[b],
    and of them those above p - window (window > 0); one that sees none gets zeros.  `max_q` and
    `max_kv`: the most new tokens and the most keys of a sequence, as far as known (0: as many keys
    as the table reaches); they are for speed alone.  `out` keeps its rows
    behind the last sequence's tokens.  A `workspace` holds partial results: calls that may run at
    the same time need one each."""
    T, dev = q.shape[0] if isinstance(q, torch.Tensor) and q.dim() == 3 else 0, _device()
    if max_q is None:
        B = max(kv_len.shape[0], 1) if isinstance(kv_len, torch.Tensor) and kv_len.dim() else 1
        max_q = -(-T // B)
    if not (0 <= max_q <= _INT and 0 <= max_kv <= _INT and 0 <= window <= _INT):
        raise ValueError(f"max_q {max_q}, max_kv {max_kv}, window {window}: each from 0 to {_INT}")
    cache, _, D, batch = _paged(k_cache, v_cache, page_table, q_start, kv_len, T, max_q, max_kv, dev)
    qt = _tokens(q, "q", 0, D, T, dev)
    Hq = q.shape[1]
    if out is None:
        out = _result(q)
        ot = _lib.Tokens.pack(out.data_ptr(), Hq * D, D)
    else:
        ot = _tokens(out, "out", Hq, D, T, dev)
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    lib = _lib.load()
    ws, room = None, 0
    if workspace is not None:
        if workspace.get_device() != dev:
            raise _elsewhere(workspace, "workspace", dev)
        if not workspace.is_contiguous():
            raise ValueError("workspace: tensor must be contiguous")
        ws, room = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    else:
        need = lib.pk_paged_attention_workspace_size(Hq, cache, batch)
        if need:
            workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
            ws, room = workspace.data_ptr(), need
    check(lib.launch_paged_attention(qt, ot, Hq, cache, batch, scale, causal, window, ws, room, _stream()),
          "launch_paged_attention")
    return out


def quantize_per_channel(w: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """quant_golden.quantize_per_channel (quant_golden.py:71-83), bit-exact."""
    K, N = w.shape
    wq = torch.empty(K, N, dtype=torch.int8, device=w.device)
    scale = torch.empty(N, dtype=torch.float32, device=w.device)
    check(_lib.load().launch_quantize_int8_per_channel(_dev(w, bf16, "w"), _dev(wq, torch.int8, "wq"),
                                                       _dev(scale, torch.float32, "scale"), K, N,
                                                       _stream()), "launch_quantize_int8_per_channel")
    return wq, scale


def matmul_int8(a: torch.Tensor, wq: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """quant_golden.matmul_int8 (quant_golden.py:91-101)."""
    K = a.shape[-1]
    M, N = a.numel() // K, wq.shape[1]
    out = torch.empty(*a.shape[:-1], N, dtype=bf16, device=a.device)
    check(_lib.load().launch_matmul_int8(_dev(a, bf16, "a"), _dev(wq, torch.int8, "wq"),
                                         _dev(scale, torch.float32, "scale"), _dev(out, bf16, "out"),
                                         M, N, K, _stream()), "launch_matmul_int8")
    return out


def int8_default_config(M: int, N: int, K: int) -> Optional[dict]:
    """Configuration launch_matmul_int8 picks for a shape (None: generic kernel)."""
    cfg = _lib.Config()
    rc = _lib.load().pk_int8_default_config(M, N, K, cfg)
    if rc == _lib.PK_ERR_UNSUPPORTED:
        return None
    check(rc, "pk_int8_default_config")
    return cfg.as_dict()


def matmul_int8_ex(epi: int, a: torch.Tensor, wq: torch.Tensor, scale: torch.Tensor,
                   residual: Optional[torch.Tensor] = None, config: Optional[dict] = None) -> torch.Tensor:
    """int8 matmul with an explicit epilogue (0 none, 1 GELU, 2 + residual) and
    launch configuration (tuning/test hook pk_matmul_int8_ex)."""
    K = a.shape[-1]
    M, N = a.numel() // K, wq.shape[1]
    out = torch.empty(*a.shape[:-1], N, dtype=bf16, device=a.device)
    cfg = None if config is None else _lib.Config(**config)
    check(_lib.load().pk_matmul_int8_ex(epi, _dev(a, bf16, "a"), _dev(wq, torch.int8, "wq"),
                                        _dev(scale, torch.float32, "scale"), _dev(out, bf16, "out"),
                                        _opt(residual, bf16, "residual"), M, N, K, cfg, None, 0,
                                        _stream()), "pk_matmul_int8_ex")
    return out


def decode_mlp_int8(x, w1q, s1, w2q, s2, workspace: Optional[torch.Tensor] = None):
    """add(matmul_int8(gelu(matmul_int8(x, W1q, s1)), W2q, s2), x) (config-5 chain)."""
    d = x.shape[-1]
    M = x.numel() // d
    F = w1q.shape[1]
    lib = _lib.load()
    need = lib.pk_decode_mlp_int8_workspace_size(M, d, F)
    if workspace is None:
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=x.device)
    out = torch.empty_like(x)
    check(lib.launch_decode_mlp_int8(_dev(x, bf16, "x"), _dev(w1q, torch.int8, "w1q"),
                                     _dev(s1, torch.float32, "s1"), _dev(w2q, torch.int8, "w2q"),
                                     _dev(s2, torch.float32, "s2"), _dev(out, bf16, "out"), M, d, F,
                                     workspace.data_ptr(), workspace.numel(), _stream()),
          "launch_decode_mlp_int8")
    return out
