"""A mixture-of-experts layer for a few tokens (``csrc/moe_few.cu``): routing and expert products without gathered or
padded rows, for decode steps.  No gradients; ``models/moe.py::moe_ffn`` picks this path or the grouped GEMMs.

The decode steps of a mixture-of-experts model are what the reference leaves to vLLM's fused expert kernels
(skyrl/backends/skyrl_train/inference_servers/vllm_worker.py).
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib

MAX_EXPERTS = 1024
MAX_TOP_K = 16
MAX_ENTRIES = 2048  # tokens x top_k of one call
_cfg_done = False


def _k():
    global _cfg_done
    lib = _lib.kernels()
    if not _cfg_done:
        vp, ci, cl = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong
        lib.sb_moe_few_route.argtypes = [vp, cl, vp, vp, vp, vp, ci, ci, ci, ci, ci, vp]
        lib.sb_moe_few_experts.argtypes = [vp, cl, vp, vp, vp, vp, vp, vp, ci, ci, ci, ci, ci, vp]
        _cfg_done = True
    return lib


def supports(T: int, num_experts: int, top_k: int, H: int, F: int) -> bool:
    """Whether the kernels take a layer of these sizes."""
    return (T * top_k <= MAX_ENTRIES and num_experts <= MAX_EXPERTS and 1 <= top_k <= min(MAX_TOP_K, num_experts)
            and H % 8 == 0 and F % 8 == 0)


def _aligned(*ts: torch.Tensor) -> bool:
    return all(t.data_ptr() % 16 == 0 for t in ts)


def _rows(h: torch.Tensor) -> tuple[torch.Tensor, int]:
    """Rows that the kernels can read 16 bytes at a time, and their stride (of a single row: any that fits)."""
    T, H = h.shape
    ok = h.stride(1) == 1 and (T == 1 or (h.stride(0) % 8 == 0 and h.stride(0) >= H)) and _aligned(h)
    if not ok:
        h = torch.empty_like(h, memory_format=torch.contiguous_format).copy_(h)
    return h, h.stride(0) if T > 1 else H


def _check_common(what, h, a, b):
    if torch.is_grad_enabled() and (h.requires_grad or a.requires_grad or b.requires_grad):
        raise ValueError(f"{what} has no gradient: call it under torch.no_grad() (moe_ffn trains)")
    dt, dev = h.dtype, h.get_device()  # -1 on the CPU
    if h.dim() != 2 or a.dtype != dt or b.dtype != dt or a.get_device() != dev or b.get_device() != dev:
        raise ValueError(f"{what}: rows [T, H] and weights must have one type and device")
    if not a.is_contiguous() or not b.is_contiguous():
        raise ValueError(f"{what}: weights must be contiguous")
    if dev >= 0 and (dt != torch.bfloat16 or h.shape[1] % 8):
        raise ValueError(f"{what}: CUDA rows must be bf16 with a width that is a multiple of 8, got {dt} [{h.shape[1]}]")
    if dev >= 0 and not _aligned(a, b):
        raise ValueError(f"{what}: weights must start on a 16-byte boundary")
    return dev


def route_few(h: torch.Tensor, router_w: torch.Tensor, top_k: int, norm_topk_prob: bool = True,
              live: torch.Tensor | None = None):
    """``(weights fp32, expert ids int32)``, both ``[T, top_k]``, largest first and ties to the lower expert:
    softmax of ``h @ router_w^T`` over the experts, renormalised over the chosen ones with ``norm_topk_prob``.

    ``live`` (``[T]`` int32): rows where it is 0 are not routed; they get id -1 and weight 0, so that the expert layer
    reads no weights for them.  A row with a NaN logit gets weights of NaN and valid ids."""
    what = "route_few"
    dev = _check_common(what, h, router_w, router_w)
    T, H = h.shape
    if router_w.dim() != 2 or router_w.shape[1] != H:
        raise ValueError(f"{what}: router weights {tuple(router_w.shape)} do not fit rows of width {H}")
    E = router_w.shape[0]
    if not 1 <= top_k <= min(MAX_TOP_K, E) or E > MAX_EXPERTS:
        raise ValueError(f"{what}: top {top_k} of {E} experts is out of range (at most {MAX_TOP_K} of {MAX_EXPERTS})")
    if live is not None and (live.dim() != 1 or live.numel() != T or live.dtype != torch.int32 or live.get_device() != dev
                             or not live.is_contiguous()):
        raise ValueError(f"{what}: live must be a contiguous int32 [{T}] tensor on the rows' device")
    if dev < 0:
        z = h.double() @ router_w.double().t()
        bad = torch.isnan(z).any(-1)
        z = torch.where(torch.isnan(z), torch.full_like(z, float("-inf")), z)
        top, idx = torch.sort(z, dim=-1, descending=True, stable=True)
        top, idx = top[:, :top_k], idx[:, :top_k].to(torch.int32)
        w = torch.exp((top - top[:, :1]).float())
        w = w / (w.sum(-1, keepdim=True) if norm_topk_prob else torch.exp((z - top[:, :1]).float()).sum(-1, keepdim=True))
        w = torch.where(bad[:, None], torch.full_like(w, float("nan")), w)
        if live is not None:
            off = (live == 0)[:, None]
            w, idx = torch.where(off, torch.zeros_like(w), w), torch.where(off, torch.full_like(idx, -1), idx)
        return w, idx
    w = h.new_empty((T, top_k), dtype=torch.float32)
    idx = torch.empty_like(w, dtype=torch.int32)
    if T == 0:
        return w, idx
    h, stride = _rows(h)
    code = _lib.call_on(dev, _k().sb_moe_few_route, h.data_ptr(), stride, router_w.data_ptr(),
                        None if live is None else live.data_ptr(), w.data_ptr(), idx.data_ptr(), T, E, H, top_k,
                        bool(norm_topk_prob))
    _lib.check(code, "sb_moe_few_route")
    return w, idx


def expert_ffn_few(h: torch.Tensor, w: torch.Tensor, idx: torch.Tensor, wgu: torch.Tensor, wd: torch.Tensor) -> torch.Tensor:
    """``out[t] = sum_s w[t, s] * wd[e] @ (silu(wg[e] @ h[t]) * (wu[e] @ h[t]))`` with ``e = idx[t, s]`` and
    ``wgu[e] = [wg; wu]``.  ``h`` ``[T, H]``, ``w`` fp32 / ``idx`` int32 ``[T, k]``, ``wgu`` ``[E, 2F, H]``, ``wd``
    ``[E, H, F]``; at most 2048 ``(t, s)`` pairs.  A slot whose id lies outside ``[0, E)`` contributes nothing (a row
    without valid slots is zero); an expert may appear in several slots of a row."""
    what = "expert_ffn_few"
    dev = _check_common(what, h, wgu, wd)
    T, H = h.shape
    if wgu.dim() != 3 or wd.dim() != 3 or wgu.shape[1] != 2 * wd.shape[2] or wgu.shape[2] != H or wd.shape[:2] != (wgu.shape[0], H):
        raise ValueError(f"{what}: weights {tuple(wgu.shape)}, {tuple(wd.shape)} do not fit rows of width {H}")
    E, F = wgu.shape[0], wd.shape[2]
    if idx.dim() != 2 or idx.shape[0] != T or w.shape != idx.shape or idx.dtype != torch.int32 or w.dtype != torch.float32:
        raise ValueError(f"{what}: weights and ids must be fp32 and int32 [{T}, k] tensors")
    if not idx.is_contiguous() or not w.is_contiguous() or idx.get_device() != dev or w.get_device() != dev:
        raise ValueError(f"{what}: weights and ids must be contiguous and on the rows' device")
    if w.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what} has no gradient: call it under torch.no_grad() (moe_ffn trains)")
    k = idx.shape[1]
    if k < 1 or T * k > MAX_ENTRIES or E > MAX_EXPERTS or F < 1:
        raise ValueError(f"{what}: {T} x {k} entries over {E} experts are out of range (at most {MAX_ENTRIES} over {MAX_EXPERTS})")
    if dev < 0:
        out = torch.zeros(T, H, dtype=torch.float32)
        y = torch.zeros(T * k, H, dtype=torch.float32)
        flat = idx.reshape(-1).long()
        for e in flat.unique().tolist():
            if not 0 <= e < E:
                continue
            at = torch.nonzero(flat == e)[:, 0]
            gu = h[at // k].float() @ wgu[e].float().t()
            act = (torch.nn.functional.silu(gu[:, :F]) * gu[:, F:]).to(h.dtype)
            y[at] = act.float() @ wd[e].float().t()
        on = ((idx >= 0) & (idx < E))[..., None]
        terms = torch.where(on, y.view(T, k, H) * w[..., None], torch.zeros(()))
        return out.add_(terms.sum(1)).to(h.dtype)
    if F % 8:
        raise ValueError(f"{what}: the experts' width must be a multiple of 8 on CUDA, got {F}")
    out = torch.empty_like(h, memory_format=torch.contiguous_format)
    if T == 0:
        return out
    h, stride = _rows(h)
    act = h.new_empty(T * k * F)
    code = _lib.call_on(dev, _k().sb_moe_few_experts, h.data_ptr(), stride, w.data_ptr(), idx.data_ptr(), wgu.data_ptr(),
                        wd.data_ptr(), act.data_ptr(), out.data_ptr(), T, k, E, H, F)
    _lib.check(code, "sb_moe_few_experts")
    return out
