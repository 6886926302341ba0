"""Mixture-of-experts FFN (Qwen3-MoE style: softmax router, top-k, optional renormalisation).

Tokens are sorted by expert so that each expert's rows are contiguous and every expert runs the
same three tcgen05 GEMM products as a dense FFN on its slice; the expert-parallel variant (dispatch
and combine over peer memory) lives in ``skyrl_b200.parallel.expert_parallel``.  Reference: the
Megatron MoE layer configured at skyrl/backends/skyrl_train/workers/megatron/megatron_worker.py:377-545
(``moe_token_dispatcher_type="alltoall"``, ``moe_grouped_gemm``).
"""

from __future__ import annotations

import torch

from ..ops import elementwise as ew
from ..ops import gemm  # noqa: F401
from ..ops import grouped_gemm as gg
from ..ops import moe_few

# Up to this many rows an expert in the mean, and without gradients, the layer runs on ``ops/moe_few.py`` unless the caller
# rules it out.  Layer times there / through the grouped GEMMs in us: 128 experts of 2048 x 768, top 8: 191 / 362 at 64
# tokens (4 rows), 342 / 369 at 256 (16 rows); 8 experts of 2048 x 4096, top 2: 114 / 164 at 64 tokens (16 rows), 178 / 154
# at 128 (32 rows).  Narrow layers at 16 rows: 104 experts of 552 x 560, top 7: 113 / 140; 64 of 256 x 256, top 4: 52 / 58.
FEW_ROWS = 16


class _RouteFn(torch.autograd.Function):
    """softmax -> top-k -> (re)normalise in one kernel per direction (``csrc/moe.cu``)."""

    @staticmethod
    def forward(ctx, logits, top_k, norm):
        import ctypes

        from ..ops import _lib

        lib = _lib.kernels()
        if not getattr(lib.sb_moe_route, "_configured", False):
            vp, ci = ctypes.c_void_p, ctypes.c_int
            lib.sb_moe_route.argtypes = [vp, vp, vp, ci, ci, ci, ci, vp]
            lib.sb_moe_route_bwd.argtypes = [vp, vp, vp, vp, vp, ci, ci, ci, ci, vp]
            lib.sb_moe_route.restype = lib.sb_moe_route_bwd.restype = ci
            lib.sb_moe_route._configured = True
        T, E = logits.shape
        logits = logits.contiguous()
        w = torch.empty((T, top_k), device=logits.device, dtype=torch.float32)
        idx = torch.empty((T, top_k), device=logits.device, dtype=torch.int32)
        _lib.check(lib.sb_moe_route(logits.data_ptr(), w.data_ptr(), idx.data_ptr(), T, E, top_k, int(norm), _lib.stream_ptr()),
                   "sb_moe_route")
        ctx.save_for_backward(logits, w, idx)
        ctx.norm, ctx.lib = bool(norm), lib
        ctx.mark_non_differentiable(idx)
        return w, idx

    @staticmethod
    def backward(ctx, dw, _didx):
        from ..ops import _lib

        logits, w, idx = ctx.saved_tensors
        T, E = logits.shape
        dlogits = torch.empty_like(logits)
        dw = dw.float().contiguous()
        _lib.check(ctx.lib.sb_moe_route_bwd(logits.data_ptr(), w.data_ptr(), idx.data_ptr(), dw.data_ptr(), dlogits.data_ptr(),
                                            T, E, idx.shape[1], int(ctx.norm), _lib.stream_ptr()), "sb_moe_route_bwd")
        return dlogits, None, None


def route_topk(h: torch.Tensor, router_w: torch.Tensor, top_k: int, norm_topk_prob: bool):
    """Returns (weights [T, k] fp32, expert ids [T, k]); router math in fp32 like the reference config."""
    logits = h.float() @ router_w.float().t()
    if logits.is_cuda and logits.shape[1] <= 1024 and top_k <= 16:
        w, idx = _RouteFn.apply(logits, top_k, norm_topk_prob)
        return w, idx.long()
    probs = torch.softmax(logits, dim=-1)
    w, idx = torch.topk(probs, top_k, dim=-1)
    if norm_topk_prob:
        w = w / w.sum(dim=-1, keepdim=True)
    return w, idx


def _takes_few(h, router_w, wgu, wd, top_k) -> bool:
    if not h.is_cuda or h.shape[0] * top_k > FEW_ROWS * wgu.shape[0] or h.dtype != torch.bfloat16:
        return False
    if torch.is_grad_enabled() and any(t.requires_grad for t in (h, router_w, wgu, wd)):
        return False
    if not all(t.dtype == h.dtype and t.is_contiguous() and t.data_ptr() % 16 == 0 for t in (router_w, wgu, wd)):
        return False
    return moe_few.supports(h.shape[0], wgu.shape[0], top_k, h.shape[1], wd.shape[2])


def moe_ffn(h: torch.Tensor, router_w: torch.Tensor, wgu: torch.Tensor, wd: torch.Tensor, top_k: int,
            norm_topk_prob: bool = True, routed_indices: torch.Tensor | None = None, layer: int | None = None, qat=None,
            live: torch.Tensor | None = None, few_tokens: bool = True) -> torch.Tensor:
    """``h``: [T, H]; ``wgu``: [E, 2F, H]; ``wd``: [E, H, F].  ``routed_indices`` replays rollout-time routing;
    with ``layer`` given, an active ``router_replay`` context records or overrides the choice.  ``live`` ([T] int32):
    rows whose result is not used where it is 0; on the path for few tokens they read no expert and come out zero.
    ``few_tokens=False`` keeps a small batch on the grouped GEMMs.  The two paths round at different places and may order
    near ties differently, so log-probabilities that meet a training forward's are computed that way."""
    T, H = h.shape
    E = wgu.shape[0]
    quantised = qat is not None and qat.enabled and torch.is_grad_enabled()
    few = few_tokens and not quantised and _takes_few(h, router_w, wgu, wd, top_k)
    if few:
        w, idx = moe_few.route_few(h, router_w, top_k, norm_topk_prob, live=live)
    else:
        w, idx = route_topk(h, router_w, top_k, norm_topk_prob)
    if layer is not None and routed_indices is None:
        from . import router_replay

        if router_replay.active():  # else no cast between the routing kernel and those that start beside its end
            routed_indices = router_replay.on_route(layer, idx.long())
    if routed_indices is not None:
        probs = torch.softmax(h.float() @ router_w.float().t(), dim=-1)
        idx = routed_indices.long()
        w = probs.gather(-1, idx.clamp_min(0) if few else idx)  # a dead row without a replayed choice keeps its -1
        if norm_topk_prob:
            w = w / w.sum(dim=-1, keepdim=True)
    if few:
        return moe_few.expert_ffn_few(h, w.float().contiguous(), idx.to(torch.int32).contiguous(), wgu, wd)
    plan = gg.plan_groups(idx.reshape(-1), E, top_k)
    # rows grouped by expert, every expert's range padded to whole 128-row tiles (padding rows are zero)
    x = gg.dispatch_rows(h, plan)
    w1, w2 = wgu, wd
    if quantised:  # fake-INT4 expert weights, straight-through
        from .qat import fake_int4

        w1 = fake_int4(w1, qat.group_size, True, qat.scale_divisor, qat.q_min)
        w2 = fake_int4(w2, qat.group_size, True, qat.scale_divisor, qat.q_min)
        # the fp32 gradient buffers belong to the parameters, not to the quantised copies
        for q, prm in ((w1, wgu), (w2, wd)):
            mg = getattr(prm, "main_grad", None)
            if mg is not None:
                q.main_grad = mg
    gu = gg.grouped_linear(x, w1, plan)
    y = gg.grouped_linear(ew.swiglu(gu), w2, plan)
    return gg.combine_rows(y, w, plan)
