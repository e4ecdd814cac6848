"""`prompt_attention` -- exact causal attention over whole prompts packed one behind the other, over the gfx950 C ABI
(mp_prompt_attention).  The role of FlashInfer's prefill in front of the reference's LSHSparseAttnServer.fill
(models/attnserver.py:112-175), for any number of prompts in one launch."""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _lib as L


def differentiated(t: torch.Tensor) -> bool:
    """Whether autograd follows t, backwards or forwards (a tangent of an open dual level)."""
    return (t.requires_grad and torch.is_grad_enabled()) or (
        forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None)


def rows_strides(t: torch.Tensor, heads: int, head_dim: int, name: str):
    """Checks a bf16 CUDA tensor [tokens, heads, head_dim] whose dims are contiguous; returns its tokens, token and head
    stride (the strides of an axis of length 1, which torch leaves arbitrary, as if it were contiguous)."""
    try:      # the common case first (the host's share of a small call is larger than the kernel's)
        n, h, d = t.shape
        if t.dtype is torch.bfloat16 and h == heads and d == head_dim and t.is_cuda:
            st, sh, sd = t.stride()
            if sd == 1 and not differentiated(t):
                return n, st if n > 1 else heads * head_dim, sh if heads > 1 else head_dim
    except (AttributeError, ValueError):
        pass
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor")
    if t.dtype is not torch.bfloat16:
        raise TypeError(f"{name}: expected dtype {torch.bfloat16}, got {t.dtype}")
    if t.dim() != 3 or t.shape[1] != heads or t.shape[2] != head_dim:
        raise ValueError(f"{name}: expected shape (tokens, {heads}, {head_dim}), got {tuple(t.shape)}")
    if not t.is_cuda:
        raise ValueError(f"{name}: expected a CUDA tensor")
    if t.stride(2) != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    raise ValueError(f"{name}: requires a gradient or has a tangent, and there is no backward (torch.no_grad() for inference)")


def written(t: torch.Tensor, dtype, shape, name: str) -> None:
    """Checks a contiguous tensor that a call is to fill."""
    L.expect(t, dtype, shape, name)
    if differentiated(t):
        raise ValueError(f"{name}: requires a gradient or has a tangent, and there is no backward")


def same_device(index: int, **tensors) -> None:
    for name, t in tensors.items():
        if t.get_device() != index:
            raise ValueError(f"{name}: on {t.device}, expected cuda:{index}")


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, scale: float | None = None,
                     out: torch.Tensor | None = None, lse: torch.Tensor | None = None):
    """q bf16 [T, H, D]; k, v bf16 [T, Hkv, D] (any token / head strides that are multiples of 8 elements: slices of one
    fused projection go in as they are); cu_seqlens int32 [B + 1]: sequence b is the rows cu_seqlens[b] .. cu_seqlens[b + 1].
    Returns (out bf16 [T, H, D], lse f32 [T, H], base 2): token i of a sequence attends to its tokens 0 .. i, query head h to
    kv head h // (H // Hkv).  scale: default head_dim ** -0.5.  Rows outside every sequence are not written: give `out` /
    `lse` where their contents matter (`out` may be q itself; any other overlap is refused).  head_dim 64 or 128.  Sums are f32, the weights are rounded to bf16 for the product with v.
    Runs on torch's current stream of q's device."""
    if not isinstance(q, torch.Tensor) or q.dim() != 3:
        raise ValueError("q: expected a tensor [tokens, heads, head_dim]")
    if not isinstance(k, torch.Tensor) or k.dim() != 3:
        raise ValueError("k: expected a tensor [tokens, heads, head_dim]")
    _, H, D = q.shape
    Hkv = k.shape[1]
    T, qt, qh = rows_strides(q, H, D, "q")
    (Tk, kt, kh), (Tv, vt, vh) = rows_strides(k, Hkv, D, "k"), rows_strides(v, Hkv, D, "v")
    if Tk != T or Tv != T:
        raise ValueError(f"k, v: expected {T} tokens, got {Tk} and {Tv}")
    if not isinstance(cu_seqlens, torch.Tensor) or cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 2:
        raise ValueError("cu_seqlens: expected a tensor [sequences + 1]")
    L.expect(cu_seqlens, torch.int32, cu_seqlens.shape, "cu_seqlens")
    if out is None:
        out = q.new_empty((T, H, D))
    else:
        written(out, torch.bfloat16, (T, H, D), "out")
    if lse is None:
        lse = q.new_empty((T, H), dtype=torch.float32)
    else:
        written(lse, torch.float32, (T, H), "lse")
    device = q.get_device()
    same_device(device, k=k, v=v, cu_seqlens=cu_seqlens, out=out, lse=lse)
    args = (q.data_ptr(), qt, qh, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, cu_seqlens.data_ptr(), cu_seqlens.shape[0] - 1, T,
            H, Hkv, D, D ** -0.5 if scale is None else float(scale), out.data_ptr(), lse.data_ptr(), L.stream_on(device))
    if device == torch.cuda.current_device():
        L.check(L.lib().mp_prompt_attention(*args))
    else:
        with torch.cuda.device(device):                  # no handle: launch where the data is
            L.check(L.lib().mp_prompt_attention(*args))
    return out, lse
