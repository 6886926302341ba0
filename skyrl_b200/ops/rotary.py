"""Rotary positions in their layouts, norms of query and key heads with the rotation in the same pass, and the serving
form that also writes keys and values to the paged cache (``csrc/qk_rope.cu``).

All three work on packed projection rows ``[T, heads * head_dim]`` (queries, then keys, then values) with int32 positions
``[T]`` and the cos | sin table of ``elementwise.build_rope_table``.  The table's width is the rotated part of a head:
elements behind it pass unchanged.  ``interleaved`` pairs neighbours ``(2i, 2i + 1)``; otherwise pairs are
``(i, i + R / 2)``.  bf16, fp16 and fp32 rows; statistics and sums in fp32, one rounding per result.  A position outside
the table gives NaN in the rotated elements.

CUDA tensors run the kernels; CPU tensors run the PyTorch formulation below.  Reference behaviour: the attention modules
that the reference runs under FSDP (skyrl/backends/skyrl_train/workers/model_wrapper.py:329-333).
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib

_DTYPE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_MAX_HEAD_DIM = 512
_cfg_done = False


def _k():
    global _cfg_done
    lib = _lib.kernels()
    if not _cfg_done:
        vp, ci, cf, cl = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_longlong
        lib.sb_qk_rope_fwd.argtypes = [vp] * 9 + [cl] * 4 + [ci] * 10 + [cf, cf, vp]
        lib.sb_qk_norm_rope_bwd_parts.argtypes = [ci, ci, ci]
        lib.sb_qk_norm_rope_bwd.argtypes = [vp] * 10 + [ci] + [cl] * 3 + [ci] * 10 + [cf, vp]
        _cfg_done = True
    return lib


# ----------------------------------------------------------------------------- checks
def _check(rows, pos, table, nq, nk, head_dim, q_norm, k_norm, what):
    T, W = rows.shape[-2:]
    if nq < 0 or nk < 0 or nq + nk < 1 or head_dim < 1 or W % head_dim or W < (nq + nk) * head_dim:
        raise ValueError(f"{what}: rows of width {W} do not hold {nq} + {nk} rotated heads of size {head_dim}")
    if head_dim > _MAX_HEAD_DIM:
        raise ValueError(f"{what}: head size {head_dim} is above {_MAX_HEAD_DIM}")
    if table.dim() != 2 or table.dtype != torch.float32 or not table.is_contiguous():
        raise ValueError(f"{what}: the rope table must be a contiguous fp32 [positions, rotated width] tensor")
    n_pos, R = table.shape
    if R < 2 or R % 2 or R > head_dim or n_pos < 1:
        raise ValueError(f"{what}: rope table {tuple(table.shape)} does not fit heads of size {head_dim}")
    if pos.dtype != torch.int32 or pos.dim() != 1 or pos.numel() != T or not pos.is_contiguous():
        raise ValueError(f"{what}: positions must be a contiguous int32 [{T}] tensor, got {pos.dtype} {tuple(pos.shape)}")
    dev = rows.get_device()  # -1 on the CPU
    if pos.get_device() != dev or table.get_device() != dev:
        raise ValueError(f"{what}: rows, positions and table must be on one device")
    if (q_norm is None) != (k_norm is None):
        raise ValueError(f"{what}: q_norm and k_norm go together")
    if q_norm is not None:
        for w in (q_norm, k_norm):
            if w.dim() != 1 or w.numel() != head_dim or not w.is_contiguous() or w.get_device() != dev:
                raise ValueError(f"{what}: norm weights must be contiguous [{head_dim}] tensors on the rows' device")


def _check_rows(x, what):
    if x.dim() != 2:
        raise ValueError(f"{what}: rows must be [T, heads * head_dim], got {tuple(x.shape)}")
    if x.dtype not in _DTYPE:
        raise ValueError(f"{what}: rows must be bf16, fp16 or fp32, got {x.dtype}")


def _is_row_major(x: torch.Tensor) -> bool:
    W = x.shape[1]
    return (x.stride(1) == 1 or W == 1) and (x.stride(0) >= W or x.shape[0] <= 1)


def _row_major(x: torch.Tensor) -> torch.Tensor:
    """Rows that the kernels can walk: unit stride inside a row, no two rows on the same memory."""
    return x if _is_row_major(x) else x.contiguous()


def _share_memory(x: torch.Tensor, out: torch.Tensor) -> bool:
    """Whether ``out`` overlaps ``x`` without being the same rows (columns of one buffer beside each other do not)."""
    def end(t):
        return t.data_ptr() + ((t.shape[-2] - 1) * t.stride(-2) + t.shape[-1]) * t.element_size()

    if out.shape[0] == 0 or out.get_device() != x.get_device():
        return False
    if x.dim() == 3:
        return x.data_ptr() < end(out) and out.data_ptr() < end(x[-1])
    if out.data_ptr() == x.data_ptr():
        return not _is_row_major(x) or (x.shape[0] > 1 and out.stride(0) != x.stride(0))
    if not _is_row_major(x) or out.data_ptr() >= end(x) or x.data_ptr() >= end(out):  # the first: read from a copy
        return False
    if x.shape[0] == 1 or out.stride(0) != x.stride(0):
        return True
    W, step = x.shape[1], x.stride(0)
    between = (out.data_ptr() - x.data_ptr()) // x.element_size() % step
    return between < W or step - between < W


# ----------------------------------------------------------------------------- PyTorch formulation
def _angles_ref(pos, table):
    known = (pos >= 0) & (pos < table.shape[0])
    cs = table[torch.where(known, pos, torch.zeros_like(pos)).long()]
    cs = torch.where(known[:, None], cs, torch.full_like(cs, float("nan")))
    return cs[:, None, : table.shape[1] // 2], cs[:, None, table.shape[1] // 2 :]


def _rotate_ref(x, cos, sin, interleaved):
    """``x``: fp32 ``[T, heads, D]``."""
    R = 2 * cos.shape[-1]
    if interleaved:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        rot = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = x[..., : R // 2], x[..., R // 2 : R]
        rot = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([rot, x[..., R:]], dim=-1)


def _fwd_ref(x, q_norm, k_norm, pos, table, nq, nk, D, eps, interleaved, sign):
    T = x.shape[0]
    cos, sin = _angles_ref(pos, table)
    h = x.reshape(T, x.shape[1] // D, D)
    parts = []
    for lo, hi, w in ((0, nq, q_norm), (nq, nq + nk, k_norm)):
        p = h[:, lo:hi].float()
        if w is not None:
            p = p * torch.rsqrt(p.pow(2).mean(-1, keepdim=True) + eps) * w.float()
        parts.append(_rotate_ref(p, cos, sin * sign, interleaved).to(x.dtype))
    return torch.cat([*parts, h[:, nq + nk :]], dim=1).flatten(1)


def _bwd_ref(dy, x, q_norm, k_norm, pos, table, nq, nk, D, eps, interleaved):
    T = x.shape[0]
    cos, sin = _angles_ref(pos, table)
    d, h = dy.reshape(T, x.shape[1] // D, D), x.reshape(T, x.shape[1] // D, D)
    dx, dws = [], []
    for lo, hi, w in ((0, nq, q_norm), (nq, nq + nk, k_norm)):
        g, p = _rotate_ref(d[:, lo:hi].float(), cos, -sin, interleaved), h[:, lo:hi].float()
        r = torch.rsqrt(p.pow(2).mean(-1, keepdim=True) + eps)
        xh = p * r
        dws.append((g * xh).sum((0, 1)))
        g = g * w.float()
        dx.append((r * (g - xh * (g * xh).mean(-1, keepdim=True))).to(x.dtype))
    return torch.cat([*dx, d[:, nq + nk :]], dim=1).flatten(1), dws[0], dws[1]


# ----------------------------------------------------------------------------- kernels
def _launch_fwd(src, dst, q_norm, k_norm, pos, table, nq, nk, D, eps, interleaved, sign, n_part=0, slots=None,
                k_cache=None, v_cache=None):
    T, W = dst.shape
    if T == 0:
        return dst
    max_pos, R = table.shape
    code = _lib.call_on(
        dst.get_device(), _k().sb_qk_rope_fwd, src.data_ptr(), dst.data_ptr(), None if q_norm is None else q_norm.data_ptr(),
        None if k_norm is None else k_norm.data_ptr(), pos.data_ptr(), table.data_ptr(),
        None if slots is None else slots.data_ptr(), None if k_cache is None else k_cache.data_ptr(),
        None if v_cache is None else v_cache.data_ptr(), 0 if k_cache is None else k_cache.shape[0] * k_cache.shape[1],
        src.stride(-2), dst.stride(0), src.stride(0) if n_part else 0, n_part, max_pos, T, nq, nk, W // D, D, R,
        _DTYPE[dst.dtype], interleaved, eps, sign)
    _lib.check(code, "sb_qk_rope_fwd")
    return dst


def _rows_like(x):
    return torch.empty_like(x, memory_format=torch.contiguous_format)


class _QKNormRopeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, q_norm, k_norm, pos, table, meta):
        ctx.meta = meta
        if x.is_cuda:
            x = _row_major(x)
            out = _launch_fwd(x, _rows_like(x), q_norm, k_norm, pos, table, *meta, 1.0)
        else:
            out = _fwd_ref(x, q_norm, k_norm, pos, table, *meta, 1.0)
        if q_norm is None:
            ctx.save_for_backward(pos, table)
        else:
            ctx.save_for_backward(pos, table, x, q_norm, k_norm)
            # taken here, not from the saved tensors: activation checkpointing hands backward detached aliases
            ctx.main_grads = (getattr(q_norm, "main_grad", None), getattr(k_norm, "main_grad", None))
        return out

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():
            raise RuntimeError("rotary / qk_norm_rope have no second derivative")
        pos, table, *rest = ctx.saved_tensors
        if not rest:
            if not dy.is_cuda:
                return _fwd_ref(dy, None, None, pos, table, *ctx.meta, -1.0), None, None, None, None, None
            dy = _row_major(dy)
            return _launch_fwd(dy, _rows_like(dy), None, None, pos, table, *ctx.meta, -1.0), None, None, None, None, None
        x, q_norm, k_norm = rest
        want, main_grads = ctx.needs_input_grad[1:3], ctx.main_grads
        if dy.is_cuda:
            dx, *dws = _launch_bwd(dy, x, q_norm, k_norm, pos, table, *ctx.meta, want, main_grads)
        else:
            dx, *dws = _bwd_ref(dy, x, q_norm, k_norm, pos, table, *ctx.meta)
        out = []
        for dw, w, mg, on in zip(dws, (q_norm, k_norm), main_grads, want):
            if not on or dw is None:
                out.append(None)
            elif mg is not None:
                mg.add_(dw)
                out.append(None)
            else:
                out.append(dw.to(w.dtype))
        return dx, *out, None, None, None


def _launch_bwd(dy, x, q_norm, k_norm, pos, table, nq, nk, D, eps, interleaved, want, main_grads):
    """Returns ``(dx, dqw, dkw)``; a weight gradient that the kernel added to its fp32 ``main_grad`` is None."""
    dy = _row_major(dy)
    T, W = x.shape
    dx = _rows_like(x)
    want_q, want_k = want
    mq, mk = main_grads[0] if want_q else None, main_grads[1] if want_k else None
    direct = mixed = False
    if mq is None and mk is None:  # stored in the weights' type
        dqw, dkw = torch.empty_like(q_norm) if want_q else None, torch.empty_like(k_norm) if want_k else None
    else:
        # added in place where every wanted gradient has its fp32 buffer; a mix goes through fp32 zeros
        direct = all(g is not None and g.is_contiguous() and g.dtype == torch.float32
                     for g, on in ((mq, want_q), (mk, want_k)) if on)
        if direct and want_q and want_k and abs(mq.data_ptr() - mk.data_ptr()) < 4 * D:
            direct = False  # one weight for queries and keys: the kernel would add to its buffer twice at once
        mixed = not direct
        dqw, dkw = (mq, mk) if direct else (torch.zeros_like(w, dtype=torch.float32) if on else None
                                            for w, on in ((q_norm, want_q), (k_norm, want_k)))
    if T == 0:
        return (dx, *(None if direct or g is None else g.zero_() for g in (dqw, dkw)))
    lib = _k()
    max_pos, R = table.shape
    heads = W // D
    part = None
    n_parts = lib.sb_qk_norm_rope_bwd_parts(T, heads, D)
    if want_q or want_k:
        part = torch.empty(n_parts * 2 * D, device=x.device, dtype=torch.float32)
    code = _lib.call_on(
        x.get_device(), lib.sb_qk_norm_rope_bwd, dy.data_ptr(), x.data_ptr(), dx.data_ptr(), q_norm.data_ptr(),
        k_norm.data_ptr(), pos.data_ptr(), table.data_ptr(), None if dqw is None else dqw.data_ptr(),
        None if dkw is None else dkw.data_ptr(), None if part is None else part.data_ptr(), n_parts, dy.stride(0), x.stride(0),
        dx.stride(0), max_pos, T, nq, nk, heads, D, R, _DTYPE[x.dtype], interleaved, direct or mixed, eps)
    _lib.check(code, "sb_qk_norm_rope_bwd")
    return (dx, None, None) if direct else (dx, dqw, dkw)


# ----------------------------------------------------------------------------- entry points
def rotary(x: torch.Tensor, pos: torch.Tensor, table: torch.Tensor, n_rot_heads: int, head_dim: int,
           interleaved: bool = False) -> torch.Tensor:
    """Rotate the first ``n_rot_heads`` heads of every row of ``x`` ``[T, heads * head_dim]``; the other heads are
    copied.  Returns new rows (``elementwise.rope`` is the in-place form for whole heads in the half layout)."""
    _check_rows(x, "rotary")
    _check(x, pos, table, n_rot_heads, 0, head_dim, None, None, "rotary")
    return _QKNormRopeFn.apply(x, None, None, pos, table, (n_rot_heads, 0, head_dim, 0.0, bool(interleaved)))


def qk_norm_rope(qkv: torch.Tensor, q_norm: torch.Tensor, k_norm: torch.Tensor, pos: torch.Tensor, table: torch.Tensor,
                 nq: int, nkv: int, head_dim: int, eps: float, interleaved: bool = False) -> torch.Tensor:
    """RMS norm of every query head (weight ``q_norm`` ``[head_dim]``) and key head (``k_norm``) of ``qkv``
    ``[T, (nq + nkv + ...) * head_dim]``, then the rotation; what lies behind the key heads is copied.  Returns new rows.
    Weight gradients go to ``main_grad`` where the weights have one; they are summed in a fixed order."""
    _check_rows(qkv, "qk_norm_rope")
    if q_norm is None or k_norm is None:
        raise ValueError("qk_norm_rope: both norm weights are needed (rotary() rotates without norms)")
    _check(qkv, pos, table, nq, nkv, head_dim, q_norm, k_norm, "qk_norm_rope")
    if q_norm.dtype != qkv.dtype or k_norm.dtype != qkv.dtype:
        raise ValueError("qk_norm_rope: norm weights must have the rows' type")
    return _QKNormRopeFn.apply(qkv, q_norm, k_norm, pos, table, (nq, nkv, head_dim, float(eps), bool(interleaved)))


def qk_rope_cache(x: torch.Tensor, pos: torch.Tensor, table: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                  slots: torch.Tensor, nq: int, nkv: int, head_dim: int, q_norm: torch.Tensor | None = None,
                  k_norm: torch.Tensor | None = None, eps: float = 1e-6, interleaved: bool = False,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """Rows of a fused QKV projection on their way into attention, in one launch and without gradients: norms (when the
    weights are given), rotation, and the key and value heads of row ``t`` written to cache slot ``slots[t]`` (a slot
    outside the cache, such as -1, writes nothing; two rows must not share a slot).

    ``x``: ``[T, (nq + 2 nkv) * head_dim]`` in the caches' type, or the fp32 partial sums ``[P, T, ...]`` of a split
    projection, which are summed (no sum's rounding shows) and rounded to that type first.  Caches: ``[blocks, block_size, nkv, head_dim]``.
    Returns the rows, in ``out`` when given; ``out`` may be ``x`` itself."""
    what = "qk_rope_cache"
    if x.dim() not in (2, 3):
        raise ValueError(f"{what}: rows must be [T, width] or partial sums [P, T, width], got {tuple(x.shape)}")
    partial = x.dim() == 3
    dt = k_cache.dtype
    if dt not in _DTYPE or v_cache.dtype != dt or x.dtype != (torch.float32 if partial else dt):
        raise ValueError(f"{what}: rows {x.dtype} and caches {dt}, {v_cache.dtype} do not go together")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, q_norm, k_norm)):
        raise ValueError(f"{what} has no gradient: use qk_norm_rope or rotary where one is needed")
    _check(x, pos, table, nq, nkv, head_dim, q_norm, k_norm, what)
    T, W = x.shape[-2:]
    if nkv < 1 or W != (nq + 2 * nkv) * head_dim:
        raise ValueError(f"{what}: rows of width {W} are not {nq} query, {nkv} key and {nkv} value heads")
    if partial and (x.shape[0] < 1 or x.stride(2) != 1 or (T > 1 and x.stride(1) < W)):
        raise ValueError(f"{what}: partial sums must be rows of unit stride")
    if q_norm is not None and (q_norm.dtype != dt or k_norm.dtype != dt):
        raise ValueError(f"{what}: norm weights must have the caches' type")
    shape = k_cache.shape
    if len(shape) != 4 or shape[2] != nkv or shape[3] != head_dim or v_cache.shape != shape:
        raise ValueError(f"{what}: caches {tuple(shape)}, {tuple(v_cache.shape)} do not hold {nkv} heads of size {head_dim}")
    if not k_cache.is_contiguous() or not v_cache.is_contiguous():
        raise ValueError(f"{what}: caches must be contiguous")
    if slots.dtype != torch.int32 or slots.dim() != 1 or slots.numel() != T or not slots.is_contiguous():
        raise ValueError(f"{what}: slots must be a contiguous int32 [{T}] tensor")
    if not (k_cache.get_device() == v_cache.get_device() == slots.get_device() == x.get_device()):
        raise ValueError(f"{what}: rows, slots and caches must be on one device")
    if out is not None and (out.shape != (T, W) or out.dtype != dt or out.get_device() != x.get_device() or out.stride(1) != 1
                            or (T > 1 and out.stride(0) < W)):
        raise ValueError(f"{what}: out must be [{T}, {W}] rows in the caches' type")
    if out is not None and _share_memory(x, out):
        raise ValueError(f"{what}: out lies on other elements of x (it may be x itself)")
    if not x.is_cuda:
        rows = x.double().sum(0).float().to(dt) if partial else x
        res = _fwd_ref(rows, q_norm, k_norm, pos, table, nq, nkv, head_dim, eps, interleaved, 1.0)
        keep = (slots >= 0) & (slots < k_cache.shape[0] * k_cache.shape[1])
        at = slots[keep].long()
        k_cache.view(-1, nkv * head_dim)[at] = res[keep, nq * head_dim : (nq + nkv) * head_dim]
        v_cache.view(-1, nkv * head_dim)[at] = res[keep, (nq + nkv) * head_dim :]
        return res if out is None else out.copy_(res)
    if not partial and (out is None or out.data_ptr() != x.data_ptr()):
        x = _row_major(x)
    if out is None:
        out = torch.empty((T, W), device=x.device, dtype=dt)
    return _launch_fwd(x, out, q_norm, k_norm, pos, table, nq, nkv, head_dim, float(eps), bool(interleaved), 1.0,
                       x.shape[0] if partial else 0, slots, k_cache, v_cache)
