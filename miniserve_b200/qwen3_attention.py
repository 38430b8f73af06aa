"""Drop-in ``Qwen3Attention`` whose per-head norm, RoPE, K/V scatter and attention are the
sm_100a kernels (src/miniserve/model/qwen3.py:65-100).

The module keeps the reference's parameter names (``qkv_proj``, ``o_proj``, ``q_norm.weight``,
``k_norm.weight``) so the reference loader (``load_weights``, model/loader.py:51-79) fills it
unchanged, and the same ``forward(x, cos, sin, k_cache, v_cache, meta)`` signature, so
``Qwen3DecoderLayer`` calls it unchanged.  The o_proj GEMM stays a library call (cuBLAS); the qkv
projection is cuBLAS followed by kernel A, or, with ``fused_qkv``, kernel E (both in one launch).
"""

from __future__ import annotations

from typing import Any

import torch
from torch import Tensor, nn

from . import _capi
from .attention import AttentionMetadata, _on_own_device, _rows, _stream, attend
from .kv_pool import HEAD_DIM, check_layer_views, is_kv8

# Smallest step (tokens) for which ``fused_qkv="auto"`` takes kernel E: measured on a B200 against
# cuBLAS + kernel A (its 16-byte form) over 28 layers, kernel E is 0.74-0.93x from 64 to 1536
# tokens, 1.01x at 2048 and 1.12-1.26x from 4096 tokens up.
FUSED_QKV_MIN_TOKENS = 2048


class HeadNorm(nn.Module):
    """Holds an RMSNorm's weight and eps (layers.py:10-22); applied inside kernel A."""

    def __init__(self, dim: int, eps: float) -> None:
        super().__init__()
        self.weight = nn.Parameter(torch.ones(dim))
        self.eps = eps


def _check_step(t: int, x: Tensor, k_cache: Tensor, num_heads: int, q_weight: Tensor, k_weight: Tensor,
                cos: Tensor, sin: Tensor, slot_mapping: Tensor, positions: Tensor | None,
                q_out: Tensor | None) -> None:
    """What kernels A and E read and write beside x's t rows fits them, on the pool's device."""
    _check_index(slot_mapping, "slot_mapping", t)
    if q_weight.numel() < HEAD_DIM or k_weight.numel() < HEAD_DIM:
        raise ValueError(f"q_norm / k_norm weights must have {HEAD_DIM} values")
    shape, sin_shape = cos.shape, sin.shape
    if shape[-1] < HEAD_DIM or sin_shape[-1] < HEAD_DIM or sin_shape[0] < shape[0]:
        raise ValueError(f"cos and sin must have rows of {HEAD_DIM} for the same positions")
    dev = k_cache.get_device()
    ok = (x.get_device() == dev and slot_mapping.get_device() == dev and q_weight.get_device() == dev
          and k_weight.get_device() == dev and cos.get_device() == dev and sin.get_device() == dev)
    if positions is not None:
        _check_index(positions, "positions", t)
        ok = ok and positions.get_device() == dev
    if q_out is not None:
        shape = q_out.shape
        if len(shape) != 3 or shape[0] < t or shape[1] != num_heads:
            raise ValueError(f"q_out must be [{t}, {num_heads}, {HEAD_DIM}]")
        ok = ok and q_out.get_device() == dev
    if not ok:
        raise ValueError(f"every argument must be on the pool's device, {k_cache.device}")


def _check_index(index: Tensor, name: str, rows: int) -> None:
    if index.dtype != torch.int64 or not index.is_contiguous():
        raise ValueError(f"{name} must be contiguous int64")
    if index.numel() < rows:
        raise ValueError(f"{rows} rows but {name} has {index.numel()} entries")


def qk_norm_rope_scatter(
    qkv: Tensor,
    q_weight: Tensor,
    k_weight: Tensor,
    eps: float,
    cos: Tensor,
    sin: Tensor,
    slot_mapping: Tensor,
    k_cache: Tensor,
    v_cache: Tensor,
    num_heads: int,
    positions: Tensor | None = None,
    q_out: Tensor | None = None,
) -> Tensor:
    """Kernel A: returns normalised, rotated q ``[T, H, 128]``; writes k (normalised, rotated)
    and v into their pool slots.  ``cos``/``sin`` are per-token rows ``[T, 128]`` fp32, or the
    whole table when ``positions`` is given (qwen3.py:94-98 + backends.py:159-160).  Into an 8-bit
    pool the rows are quantised as they are written."""
    nb, kvh = check_layer_views(k_cache, v_cache, kv8=True)
    t = int(qkv.shape[0])
    width = (num_heads + 2 * kvh) * HEAD_DIM
    if qkv.dim() != 2 or qkv.shape[1] != width or qkv.stride(1) != 1 or qkv.dtype != torch.bfloat16:
        raise ValueError(f"qkv must be bf16 [T, {width}] with unit column stride")
    if q_weight.dtype != torch.bfloat16 or k_weight.dtype != torch.bfloat16:
        raise ValueError("q_norm / k_norm weights must be bf16")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32 or cos.stride(-1) != 1:
        raise ValueError("cos/sin must be fp32 with unit column stride")
    if sin.stride(0) != cos.stride(0):
        raise ValueError("cos and sin must share a row stride")
    if positions is None and cos.shape[0] < t:
        raise ValueError("per-token cos/sin rows must cover every token")
    _check_step(t, qkv, k_cache, num_heads, q_weight, k_weight, cos, sin, slot_mapping, positions, q_out)
    if q_out is None:
        q_out = torch.empty((t, num_heads, HEAD_DIM), dtype=torch.bfloat16, device=qkv.device)
    pos_ptr, max_pos = None, 0
    if positions is not None:
        pos_ptr, max_pos = positions.data_ptr(), int(cos.shape[0])
    lib = _capi.load()
    args = (
        qkv.data_ptr(), int(qkv.stride(0)), t, num_heads, kvh, q_weight.data_ptr(),
        k_weight.data_ptr(), float(eps), cos.data_ptr(), sin.data_ptr(), int(cos.stride(0)),
        pos_ptr, max_pos, slot_mapping.data_ptr(), q_out.data_ptr(), _rows(q_out, "q_out"),
    )
    dev = qkv.device
    if is_kv8(k_cache):
        rc = _on_own_device(lib.ms_qk_norm_rope_scatter_kv8, dev, *args, k_cache.data_ptr(), nb,
                            _stream(dev))
    else:
        rc = _on_own_device(lib.ms_qk_norm_rope_scatter, dev, *args, k_cache.data_ptr(),
                            v_cache.data_ptr(), nb, _stream(dev))
    _capi.check(rc, "qk_norm_rope_scatter")
    return q_out


def qkv_proj_norm_rope_scatter(
    x: Tensor,
    w_qkv: Tensor,
    q_weight: Tensor,
    k_weight: Tensor,
    eps: float,
    cos: Tensor,
    sin: Tensor,
    slot_mapping: Tensor,
    k_cache: Tensor,
    v_cache: Tensor,
    num_heads: int,
    positions: Tensor | None = None,
    q_out: Tensor | None = None,
) -> Tensor:
    """Kernel E: ``qkv_proj`` (``x @ w_qkv.T``, qwen3.py:94) with kernel A as its epilogue, in one
    tensor-core launch.  Same outputs as ``qk_norm_rope_scatter(x @ w_qkv.T, ...)`` up to the
    GEMM's fp32 accumulation order (a projection output may differ by one bf16 ulp)."""
    nb, kvh = check_layer_views(k_cache, v_cache)
    t = int(x.shape[0])
    if x.dim() != 2 or x.stride(1) != 1 or x.dtype != torch.bfloat16:
        raise ValueError("x must be bf16 [T, hidden] with unit column stride")
    hidden = int(x.shape[1])
    width = (num_heads + 2 * kvh) * HEAD_DIM
    if (w_qkv.dim() != 2 or tuple(w_qkv.shape) != (width, hidden) or w_qkv.stride(1) != 1
            or w_qkv.dtype != torch.bfloat16):
        raise ValueError(f"w_qkv must be bf16 [{width}, {hidden}] with unit column stride")
    if q_weight.dtype != torch.bfloat16 or k_weight.dtype != torch.bfloat16:
        raise ValueError("q_norm / k_norm weights must be bf16")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32 or cos.stride(-1) != 1:
        raise ValueError("cos/sin must be fp32 with unit column stride")
    if sin.stride(0) != cos.stride(0):
        raise ValueError("cos and sin must share a row stride")
    if positions is None and cos.shape[0] < t:
        raise ValueError("per-token cos/sin rows must cover every token")
    _check_step(t, x, k_cache, num_heads, q_weight, k_weight, cos, sin, slot_mapping, positions, q_out)
    if q_out is None:
        q_out = torch.empty((t, num_heads, HEAD_DIM), dtype=torch.bfloat16, device=x.device)
    pos_ptr, max_pos = None, 0
    if positions is not None:
        pos_ptr, max_pos = positions.data_ptr(), int(cos.shape[0])
    lib = _capi.load()
    rc = _on_own_device(
        lib.ms_qkv_proj_norm_rope_scatter, x.device, x.data_ptr(), int(x.stride(0)), t, hidden, w_qkv.data_ptr(), int(w_qkv.stride(0)),
        num_heads, kvh, q_weight.data_ptr(), k_weight.data_ptr(), float(eps), cos.data_ptr(),
        sin.data_ptr(), int(cos.stride(0)), pos_ptr, max_pos, slot_mapping.data_ptr(),
        q_out.data_ptr(), _rows(q_out, "q_out"), k_cache.data_ptr(), v_cache.data_ptr(), nb,
        _stream(x.device),
    )
    _capi.check(rc, "qkv_proj_norm_rope_scatter")
    return q_out


class Qwen3Attention(nn.Module):
    """Same constructor and forward as the reference module (qwen3.py:65-100)."""

    def __init__(self, cfg: Any) -> None:
        super().__init__()
        self.num_heads = cfg.num_attention_heads
        self.num_kv_heads = cfg.num_key_value_heads
        self.head_dim = cfg.head_dim
        if self.head_dim != HEAD_DIM or self.num_heads != 2 * self.num_kv_heads:
            raise ValueError("the sm_100a path serves head_dim 128 with two query heads per KV head")
        self.q_size = self.num_heads * self.head_dim
        self.kv_size = self.num_kv_heads * self.head_dim
        self.scale = self.head_dim**-0.5
        self.qkv_proj: nn.Module = nn.Linear(cfg.hidden_size, self.q_size + 2 * self.kv_size,
                                             bias=False)
        self.o_proj: nn.Module = nn.Linear(self.q_size, cfg.hidden_size, bias=False)
        self.q_norm = HeadNorm(self.head_dim, cfg.rms_norm_eps)
        self.k_norm = HeadNorm(self.head_dim, cfg.rms_norm_eps)
        # True: kernel E computes the projection and the norm/RoPE/scatter in one launch (faster
        # from about a thousand tokens per step; a projection output can differ from cuBLAS's by
        # one bf16 ulp, from the GEMM's accumulation order).  False: cuBLAS, then kernel A.
        # "auto": kernel E for steps of at least FUSED_QKV_MIN_TOKENS tokens, else cuBLAS + A.
        fused = getattr(cfg, "fused_qkv", False)
        if fused != "auto" and not isinstance(fused, (bool, int)):
            raise ValueError(f"fused_qkv must be True, False or 'auto', not {fused!r}")
        self.fused_qkv: bool | str = fused if fused == "auto" else bool(fused)

    def forward(
        self,
        x: Tensor,
        cos: Tensor,
        sin: Tensor,
        k_cache: Tensor,
        v_cache: Tensor,
        meta: AttentionMetadata,
    ) -> Tensor:
        t = x.shape[0]
        fused = self.fused_qkv is True or (self.fused_qkv == "auto" and t >= FUSED_QKV_MIN_TOKENS)
        # Kernel E writes a bf16 pool only; an 8-bit pool takes the projection and kernel A.
        if fused and isinstance(self.qkv_proj, nn.Linear) and not is_kv8(k_cache):
            q = qkv_proj_norm_rope_scatter(
                x, self.qkv_proj.weight, self.q_norm.weight, self.k_norm.weight, self.q_norm.eps,
                cos, sin, meta.slot_mapping, k_cache, v_cache, self.num_heads,
            )
        else:
            qkv = self.qkv_proj(x)
            q = qk_norm_rope_scatter(
                qkv, self.q_norm.weight, self.k_norm.weight, self.q_norm.eps, cos, sin,
                meta.slot_mapping, k_cache, v_cache, self.num_heads,
            )
        out = attend(q, k_cache, v_cache, meta, self.scale)
        result: Tensor = self.o_proj(out.reshape(t, self.q_size))
        return result
